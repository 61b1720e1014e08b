"""Expert readout without a GPU: refusals, shapes on Meta tensors, sizes of the C ABI, construction."""

import ctypes

import pytest
import torch

from fsctep_amd import _lib, expert_ops as X
from fsctep_amd.experts import ExpertReadout


class Dims(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_int64), ("width", ctypes.c_int32), ("hidden", ctypes.c_int32),
                ("n_experts", ctypes.c_int32), ("k", ctypes.c_int32), ("dtype", ctypes.c_int32)]


def meta(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="GPU only"):
        X.rms_norm(x, w)
    with pytest.raises(RuntimeError, match="GPU only"):
        X.route_experts(x, 2)
    with pytest.raises(RuntimeError, match="GPU only"):
        X.expert_mlp(x, torch.zeros(4, 2, dtype=torch.int32), torch.ones(4, 2), torch.zeros(3, 10, 8), torch.zeros(3, 8, 5))
    with pytest.raises(ValueError, match="score"):
        X.route_experts(x, 2, score="relu")


def test_meta_shapes():
    x = meta(7, 20, dtype=torch.bfloat16)
    y, z = X.rms_norm(x, meta(20), meta(7, 20, dtype=torch.bfloat16))
    assert y.shape == z.shape == (7, 20) and y.dtype == torch.bfloat16
    q, s, _ = X.rms_norm_q8(x, meta(20))
    assert q.dtype == torch.int8 and s.shape == (7,)
    i, w = X.route_experts(meta(7, 6), 3)
    assert i.shape == w.shape == (7, 3) and i.dtype == torch.int32 and w.dtype == torch.float32
    y = X.expert_mlp(meta(7, 20), meta(7, 3, dtype=torch.int32), meta(7, 3), meta(6, 18, 20), meta(6, 20, 9))
    assert y.shape == (7, 20)


@pytest.mark.parametrize("change,msg", [
    (dict(x=(7, 20, 1)), "dimensions"), (dict(w_in=(6, 17, 20)), "w_in"), (dict(w_out=(6, 21, 9)), "w_out"),
    (dict(index=(8, 3)), "index"), (dict(weight=(7, 2)), "weight")])
def test_expert_mlp_shapes_are_checked(change, msg):
    shape = dict(x=(7, 20), index=(7, 3), weight=(7, 3), w_in=(6, 18, 20), w_out=(6, 20, 9)) | change
    with pytest.raises(RuntimeError, match=msg):
        torch.ops.fsctep.expert_mlp_forward(meta(*shape["x"]), meta(*shape["index"], dtype=torch.int32),
                                            meta(*shape["weight"]), meta(*shape["w_in"]), meta(*shape["w_out"]), False)


def test_types_are_checked():
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        X.rms_norm(meta(4, 8, dtype=torch.float16), meta(8, dtype=torch.float16))
    with pytest.raises(RuntimeError, match="weight must be float32 or of x's type"):
        X.rms_norm(meta(4, 8), meta(8, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="residual must have x's"):
        X.rms_norm(meta(4, 8), meta(8), meta(5, 8))
    with pytest.raises(RuntimeError, match="one type"):
        torch.ops.fsctep.expert_mlp_forward(meta(7, 20), meta(7, 3, dtype=torch.int32), meta(7, 3),
                                            meta(6, 18, 20, dtype=torch.bfloat16), meta(6, 20, 9), False)
    with pytest.raises(RuntimeError, match="int32"):
        torch.ops.fsctep.expert_mlp_forward(meta(7, 20), meta(7, 3, dtype=torch.int64), meta(7, 3), meta(6, 18, 20),
                                            meta(6, 20, 9), False)


def test_c_abi_refusals():
    lib = _lib.load()
    n = [ctypes.c_int64() for _ in range(4)]
    out = [ctypes.byref(v) for v in n]
    assert lib.fsc_expert_sizes(ctypes.byref(Dims(10, 20, 9, 6, 3, 0)), *out) == 0
    assert n[1].value == 30 * 2 * 16            # gate and up, hidden padded to 8
    for bad, msg in ((Dims(-1, 20, 9, 6, 3, 0), b"rows"), (Dims(10, 0, 9, 6, 3, 0), b"width"),
                     (Dims(10, 20, 9, 513, 3, 0), b"experts"), (Dims(10, 20, 9, 6, 65, 0), b"slots"),
                     (Dims(10, 20, 9, 6, 3, 7), b"float32 or bfloat16")):
        assert lib.fsc_expert_sizes(ctypes.byref(bad), *out) == 1 and msg in lib.fsc_last_error()
    assert lib.fsc_expert_sizes(None, *out) == 1
    assert lib.fsc_rms_norm_forward(4, 8, 5, 0, 8, 0, None, None, None, 1e-6, None, None, None, None) == 1
    assert b"float32 or bfloat16" in lib.fsc_last_error()
    assert lib.fsc_rms_norm_forward(4, 8, 0, 0, 8, 0, None, None, None, 1e-6, None, None, None, None) == 1
    assert b"null" in lib.fsc_last_error()
    for k, groups, kept, best, scale, msg in ((9, 1, 1, 1, 1.0, b"k must"), (2, 3, 1, 1, 1.0, b"divide"),
                                              (2, 2, 3, 1, 1.0, b"groups_kept"), (5, 2, 1, 1, 1.0, b"kept groups"),
                                              (2, 1, 1, 3, 1.0, b"group_best"), (2, 1, 1, 1, 0.0, b"scale")):
        assert lib.fsc_route_experts(4, 8, 0, 8, None, None, k, 0, groups, kept, best, 1, scale, None, None, None) == 1
        assert msg in lib.fsc_last_error(), msg


def test_zero_rows_need_no_arrays():
    lib = _lib.load()
    assert lib.fsc_rms_norm_forward(0, 8, 0, 0, 8, 0, None, None, None, 1e-6, None, None, None, None) == 0
    assert lib.fsc_route_experts(0, 8, 0, 8, None, None, 2, 0, 1, 1, 1, 1, 1.0, None, None, None) == 0


def test_readout_construction():
    m = ExpertReadout(20, 8, 4, k=2, layers=2, score="sigmoid")
    assert sorted(m.state_dict()) == sorted(f"layers.{i}.{n}" for i in range(2)
                                            for n in ("norm", "gate", "w_in", "w_out", "balance"))
    assert float(m.layers[0].w_out.detach().abs().max()) == 0
    layer = m.layers[0]
    layer.rebalance(torch.tensor([[0, 1], [0, -1], [0, 2]], dtype=torch.int32), rate=0.5)
    assert layer.balance.tolist() == [-0.5, 0.5, 0.5, 0.5]   # counts 3, 1, 1, 0
    with pytest.raises(ValueError):
        ExpertReadout(20, 8, 4, k=5)
    with pytest.raises(ValueError):
        ExpertReadout(20, 8, 4, score="relu")
    with pytest.raises(RuntimeError, match="no gradient"):
        m.to_8_bits()(torch.zeros(3, 20), differentiable=True)


def test_a_trunk_without_experts_keeps_its_parameters():
    from sparse_helpers import seeded_hip_model
    m = seeded_hip_model(32, 2, 0)
    assert m.readout_experts is None and not any("expert" in k for k in m.state_dict())
