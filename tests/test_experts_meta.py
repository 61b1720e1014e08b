"""The expert readout's operators on Meta tensors: forward-mode derivatives and arguments that the GPU refuses are refused
there too."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from fsctep_amd import expert_ops as X
from test_experts_host import meta


def mlp_args(dtype=torch.float32):
    return dict(x=meta(7, 20, dtype=dtype), index=meta(7, 3, dtype=torch.int32), weight=meta(7, 3),
                w_in=meta(6, 18, 20, dtype=dtype), w_out=meta(6, 20, 9, dtype=dtype))


FORWARD_MODE = ([("norm", n) for n in ("x", "weight", "residual")] + [("route", "logits")] +
                [("mlp", n) for n in ("x", "weight", "w_in", "w_out")] + [("norm_q8", "x")])


@pytest.mark.parametrize("op,which", FORWARD_MODE)
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(op, which, grad):
    """A tangent is not dropped, with and without grad mode."""
    args = dict(norm=dict(x=meta(7, 20), weight=meta(20), residual=meta(7, 20)), route=dict(logits=meta(7, 6), k=3),
                norm_q8=dict(x=meta(7, 20), weight=meta(20)), mlp=mlp_args())[op]
    call = dict(norm=X.rms_norm, norm_q8=X.rms_norm_q8, route=X.route_experts, mlp=X.expert_mlp)[op]
    with torch.set_grad_enabled(grad), fwd.dual_level():
        args[which] = fwd.make_dual(args[which], torch.empty_like(args[which]))
        with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward AD|Forward AD"):
            call(**args)


@pytest.mark.parametrize("change,msg", [
    (dict(x=meta(7, 20, 1)), "dimensions"), (dict(w_in=meta(6, 17, 20)), "w_in must"), (dict(w_out=meta(6, 21, 9)), "w_out must"),
    (dict(index=meta(8, 3, dtype=torch.int32)), "index must"), (dict(index=meta(7, 3, dtype=torch.int64)), "int32"),
    (dict(weight=meta(7, 2)), "weight must"), (dict(weight=meta(7, 3, dtype=torch.bfloat16)), "float32"),
    (dict(x=meta(7, 20, dtype=torch.bfloat16)), "one type"), (mlp_args(torch.float16), "float32 or bfloat16"),
    (mlp_args(torch.int8), "float32 or bfloat16"), (dict(index=meta(7, 65, dtype=torch.int32), weight=meta(7, 65)), "64 slots"),
    (dict(w_in=meta(513, 18, 20), w_out=meta(513, 20, 9)), "512 experts")])
def test_products_are_checked(change, msg):
    with pytest.raises(RuntimeError, match=msg):
        X.expert_mlp(**(mlp_args() | change))
    with pytest.raises(RuntimeError, match=msg):      # the op as a program without gradients reaches it
        with torch.inference_mode():
            X.expert_mlp(**(mlp_args() | change))
    if msg != "float32 or bfloat16":
        torch.ops.fsctep.expert_mlp(*mlp_args().values())


@pytest.mark.parametrize("change,msg", [
    (dict(k=7), "k must"), (dict(k=0), "k must"), (dict(logits=meta(7, 20), k=17), "k must"), (dict(logits=meta(7, 6, 1)), "dimensions"),
    (dict(logits=meta(7, 6, dtype=torch.float16)), "float32 or bfloat16"), (dict(logits=meta(7, 513)), "512 experts"),
    (dict(bias=meta(5)), "bias must be"), (dict(bias=meta(6, dtype=torch.bfloat16)), "bias must be float32"),
    (dict(groups=4), "divide"), (dict(groups=2, groups_kept=3), "groups_kept"), (dict(groups=3, k=3), "kept groups"),
    (dict(group_best=3), "group_best"), (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(scale=1e39), "scale")])
def test_routing_is_checked(change, msg):
    args = dict(logits=meta(7, 6), k=3) | change
    with pytest.raises(RuntimeError, match=msg):
        X.route_experts(**args)
    with pytest.raises(RuntimeError, match="score"):
        torch.ops.fsctep.route_experts(meta(7, 6), None, 3, 2 ** 32, 1, 1, 1, True, 1.0)


@pytest.mark.parametrize("change,msg", [
    (dict(codes=meta(7, 20)), "int8 codes"), (dict(scale=meta(8)), "x_scale"), (dict(w_in_scale=meta(6, 9)), "w_in_scale"),
    (dict(w_out_scale=meta(6, 20, dtype=torch.bfloat16)), "w_out_scale"), (dict(w_in=meta(6, 18, 20)), "one type"),
    (dict(weight=meta(7, 2)), "weight must")])
def test_8_bit_products_are_checked(change, msg):
    i8 = dict(dtype=torch.int8)
    args = dict(codes=meta(7, 20, **i8), scale=meta(7), index=meta(7, 3, dtype=torch.int32), weight=meta(7, 3),
                w_in=meta(6, 18, 20, **i8), w_in_scale=meta(6, 18), w_out=meta(6, 20, 9, **i8), w_out_scale=meta(6, 20))
    assert X.expert_mlp_q8(**args).dtype == torch.bfloat16
    with pytest.raises(RuntimeError, match=msg):
        X.expert_mlp_q8(**(args | change))


def test_shapes_of_sizes_a_trace_does_not_know():
    """The number of rows symbolic: one trace serves every size."""
    from torch.fx.experimental.symbolic_shapes import ShapeEnv
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(shape_env=ShapeEnv()) as mode:
        x, index, weight = (mode.from_tensor(t, symbolic_context=None) for t in (
            torch.empty(7, 20), torch.empty(7, 3, dtype=torch.int32), torch.empty(7, 3)))
        y = torch.ops.fsctep.expert_mlp(x, index, weight, torch.empty(6, 18, 20), torch.empty(6, 20, 9))
        assert y.shape == x.shape
