"""Operators of the training step without a GPU: refusals, shapes on Meta tensors, sizes of the C ABI, the optimiser's
arguments, and the 8-bit format of the oracle."""

import ctypes

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwd

from fsctep_amd import _lib, learn_ops as L, optim
from oracle import learn as O


def meta(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="meta")


OPS = ["layer_norm", "layer_norm_backward", "layer_norm_backward_twice", "embedding", "embedding_backward", "grad_norm",
       "adamw_", "adamw_q8_", "adamw_values"]


@pytest.mark.parametrize("name", OPS)
def test_ops_are_registered_in_cpp(name):
    assert getattr(torch.ops.fsctep, name).default._schema.name == f"fsctep::{name}"
    for key in ("CUDA", "Meta", "CPU"):
        assert torch._C._dispatch_has_kernel_for_dispatch_key(f"fsctep::{name}", key)


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 8)
    for call in (lambda: L.layer_norm(x), lambda: L.embedding(x, torch.zeros(3, dtype=torch.long)),
                 lambda: optim.grad_norm([x]),
                 lambda: optim.adamw_step([x], [x.clone()], [x.clone()], [x.clone()], [torch.zeros(())]),
                 lambda: optim.moment_values(torch.zeros(4, dtype=torch.uint8), torch.zeros(1))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_meta_shapes():
    y = L.layer_norm(meta(7, 20, dtype=torch.bfloat16), meta(20), meta(20), activation="silu")
    assert y.shape == (7, 20) and y.dtype == torch.bfloat16
    x, w, b = (meta(*s).requires_grad_(True) for s in ((7, 20), (20,), (20,)))
    dy = meta(7, 20).requires_grad_(True)
    dx, dw, db = torch.autograd.grad(L.layer_norm(x, w, b), (x, w, b), dy, create_graph=True)
    got = torch.autograd.grad((dx, dw, db), (x, w, b, dy), (meta(7, 20), meta(20), meta(20)))
    assert [t.shape for t in got] == [x.shape, w.shape, b.shape, dy.shape]
    t = meta(9, 6).requires_grad_(True)
    e = L.embedding(t, meta(3, 5, dtype=torch.int32), 2.0)
    assert e.shape == (3, 5, 6)
    assert torch.autograd.grad(e, t, meta(3, 5, 6))[0].shape == (9, 6)
    assert optim.grad_norm([meta(3), meta(2, 2, dtype=torch.bfloat16)]).shape == ()
    assert optim.root_values(meta(300, dtype=torch.uint8), meta(2)).shape == (300,)


@pytest.mark.parametrize("args,msg", [
    (dict(x=meta(4)), "dimensions"), (dict(x=meta(4, 8, dtype=torch.float16)), "float32 or bfloat16"),
    (dict(x=meta(4, 0), weight=None, bias=None), "width"), (dict(weight=meta(7)), "weight must be"),
    (dict(bias=meta(8, 1)), "bias must be"), (dict(weight=meta(8, dtype=torch.bfloat16)), "of x's type"),
    (dict(x=meta(4, 8, dtype=torch.bfloat16), weight=meta(8, dtype=torch.bfloat16)), "one type"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps")])
def test_layer_norm_arguments(args, msg):
    with pytest.raises(RuntimeError, match=msg):
        L.layer_norm(**(dict(x=meta(4, 8), weight=meta(8), bias=meta(8)) | args))


def test_unknown_activation():
    with pytest.raises(ValueError, match="activation"):
        L.layer_norm(meta(4, 8), activation="relu")
    with pytest.raises(RuntimeError, match="activation"):
        torch.ops.fsctep.layer_norm(meta(4, 8), None, None, 1e-5, 7, False)


@pytest.mark.parametrize("call,msg", [
    (lambda: L.embedding(meta(4, 8, 2), meta(3, dtype=torch.int64)), "table must be"),
    (lambda: L.embedding(meta(4, 8, dtype=torch.float64), meta(3, dtype=torch.int64)), "float32 or bfloat16"),
    (lambda: L.embedding(meta(4, 8), meta(3)), "int32 or int64"),
    (lambda: L.embedding(meta(4, 8), meta(3, dtype=torch.int64), float("inf")), "finite"),
    (lambda: torch.ops.fsctep.embedding(meta(4, 8), meta(3, 1, dtype=torch.int64), 1.0), "one dimension"),
    (lambda: torch.ops.fsctep.embedding_backward(meta(4, 8), meta(3, dtype=torch.int64), 9, 1.0), "tokens, width"),
    (lambda: optim.moment_values(meta(300, dtype=torch.uint8), meta(3)), "scale must be"),
    (lambda: optim.moment_values(meta(300), meta(2)), "uint8")])
def test_arguments(call, msg):
    with pytest.raises(RuntimeError, match=msg):
        call()


def test_empty_lists():
    with pytest.raises(ValueError, match="no gradients"):
        optim.grad_norm([])
    assert optim.adamw_step([], [], [], [], []) is None
    assert optim.adamw_step_q8([], [], [], [], [], [], []) is None


def step_args(n=300, dtype=torch.float32):
    return dict(params=[meta(n, dtype=dtype)], grads=[meta(n, dtype=dtype)], exp_avgs=[meta(n)], exp_avg_sqs=[meta(n)],
                steps=[meta(())])


@pytest.mark.parametrize("change,msg", [
    (dict(grads=[]), "gradients for"), (dict(grads=[meta(299)]), "parameter's shape"),
    (dict(grads=[meta(300, dtype=torch.bfloat16)]), "shape and type"), (dict(params=[meta(300, dtype=torch.float64)]), "float32 or bfloat16"),
    (dict(exp_avgs=[meta(300, dtype=torch.bfloat16)]), "first moments"), (dict(exp_avg_sqs=[meta(301)]), "second moments"),
    (dict(steps=[meta(2)]), "step counts"), (dict(steps=[meta((), dtype=torch.int64)]), "step counts"),
    (dict(params=[meta(20, 15).t()], grads=[meta(15, 20)], exp_avgs=[meta(15, 20)], exp_avg_sqs=[meta(15, 20)]), "not contiguous"),
    (dict(lr=torch.zeros((), device="meta", dtype=torch.float64)), "single float32"),
    (dict(masters=[meta(300), meta(300)]), "as many as parameters"), (step_args(dtype=torch.bfloat16), "masters"), (step_args(dtype=torch.bfloat16) | dict(masters=[meta(299)]), "master 0")])
def test_step_arguments(change, msg):
    # meta tensors have no GPU kernel's refusal of devices before these checks
    a = step_args() | change
    with pytest.raises(RuntimeError, match=msg):
        optim.adamw_step(**a)


@pytest.mark.parametrize("bad", [dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(weight_decay=-1.0),
                                 dict(lr=-1.0), dict(max_norm=0.0), dict(max_norm=float("nan")), dict(state_bits=16)])
def test_optimiser_settings(bad):
    with pytest.raises(ValueError):
        optim.AdamW([torch.zeros(3, requires_grad=True)], **bad)


@pytest.mark.parametrize("which", ["x", "weight", "bias", "table"])
def test_forward_mode_derivatives_are_refused(which):
    args = dict(x=meta(7, 20), weight=meta(20), bias=meta(20))
    with fwd.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward AD|Forward AD"):
            if which == "table":
                L.embedding(fwd.make_dual(meta(4, 8), meta(4, 8)), meta(3, dtype=torch.int64))
            else:
                args[which] = fwd.make_dual(args[which], torch.empty_like(args[which]))
                L.layer_norm(**args)


def test_third_derivatives_of_the_norm_are_refused():
    x, dy = meta(7, 20).requires_grad_(True), meta(7, 20).requires_grad_(True)
    dx, = torch.autograd.grad(L.layer_norm(x), x, dy, create_graph=True)
    gx, = torch.autograd.grad(dx.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="not implemented|does not require grad"):
        torch.autograd.grad(gx.sum(), x)


def test_optimiser_is_copied_with_its_settings():
    import copy
    p = torch.zeros(3, requires_grad=True)
    opt = copy.deepcopy(optim.AdamW([p], lr=0.5, max_norm=2.0, state_bits=8))
    assert opt.max_norm == 2.0 and opt.state_bits == 8 and opt.param_groups[0]["lr"] == 0.5 and opt.grad_norm is None


def test_train_step_wants_a_model_in_training():
    with pytest.raises(ValueError, match="train"):
        optim.train_step(torch.nn.Linear(2, 2).eval(), None, None, None, None, None, None, None)


class Adam(ctypes.Structure):
    _fields_ = [("n", ctypes.c_int64), ("dtype", ctypes.c_int32), ("pad", ctypes.c_int32)] + \
        [(k, ctypes.c_void_p) for k in ("p", "g", "m", "v", "m_scale", "v_scale", "master", "step")]


class Settings(ctypes.Structure):
    _fields_ = [(k, ctypes.c_double) for k in ("lr", "beta1", "beta2", "eps", "weight_decay", "max_norm")] + \
        [("lr_tensor", ctypes.c_void_p), ("norm", ctypes.c_void_p), ("bits", ctypes.c_int32), ("pad", ctypes.c_int32)]


def test_c_abi_of_the_step_refuses_without_a_gpu():
    """No pointer here is one: every call has to end in a check."""
    lib, one = _lib.load(), 1 << 20
    ok = dict(n=300, dtype=0, p=one, g=one, m=one, v=one, step=one)
    rule = dict(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0, max_norm=0.0, bits=32)
    for tensor, settings, msg in (
            (ok | dict(g=None), rule, b"gradient is null"), (ok | dict(p=None), rule, b"parameter or a state"),
            (ok | dict(v=None), rule, b"parameter or a state"), (ok | dict(step=None), rule, b"step count"),
            (ok | dict(dtype=1), rule, b"float32 copy"), (ok | dict(dtype=2), rule, b"float32 or bfloat16"),
            (ok | dict(n=-1), rule, b"gradient is null"), (ok | dict(n=(1 << 34) + 1), rule, b"2^34"),
            (ok, rule | dict(bits=16), b"32 or 8 bits"), (ok, rule | dict(bits=8), b"scale is null"),
            (ok, rule | dict(beta1=1.0), b"betas"), (ok, rule | dict(beta2=float("nan")), b"betas"),
            (ok, rule | dict(eps=-1.0), b"negative"), (ok, rule | dict(norm=one), b"max_norm")):
        t, s = Adam(**tensor), Settings(**settings)
        assert lib.fsc_adamw_step(1, ctypes.byref(t), ctypes.byref(s), ctypes.c_void_p(one), None) == 1
        assert msg in lib.fsc_last_error(), (msg, lib.fsc_last_error())
    t, s = Adam(**ok), Settings(**rule)
    assert lib.fsc_adamw_step(1, ctypes.byref(t), ctypes.byref(s), None, None) == 1
    assert lib.fsc_adamw_step(1, ctypes.byref(t), None, ctypes.c_void_p(one), None) == 1
    assert lib.fsc_grad_norm(1, ctypes.byref(t), None, None, None) == 1
    a, b = ctypes.c_int64(), ctypes.c_int64()
    assert lib.fsc_adamw_workspace(1, ctypes.byref(t), ctypes.byref(a), ctypes.byref(b)) == 0 and a.value > 0 and b.value == 8
    assert lib.fsc_embedding_backward((1 << 31) - 1, 1 << 20, 5, 0, 32, 0, ctypes.c_void_p(one), ctypes.c_void_p(one), 1.0,
                                      ctypes.c_void_p(one), ctypes.c_void_p(one), None) == 1
    assert b"2^41" in lib.fsc_last_error()


def test_c_abi_refuses_without_a_gpu():
    lib = _lib.load()
    n = ctypes.c_int64()
    assert lib.fsc_layer_norm_workspace(10, 128, ctypes.byref(n)) == 0 and n.value >= 2 * 128
    assert lib.fsc_layer_norm_workspace(-1, 128, ctypes.byref(n)) == 1
    assert lib.fsc_embedding_workspace(10, 128, 1 << 40, ctypes.byref(n)) == 1
    assert lib.fsc_layer_norm_forward(4, 8, 2, 0, 0, 8, None, None, None, 1e-5, None, None, None, None) == 1
    assert b"float32 or bfloat16" in lib.fsc_last_error()
    assert lib.fsc_layer_norm_forward(4, 8, 0, 0, 0, 8, None, None, None, 1e-5, None, None, None, None) == 1
    assert b"null array" in lib.fsc_last_error()
    assert lib.fsc_embedding_forward(4, 8, 3, 0, 16, 8, None, None, 1.0, None, None) == 1
    assert b"int32 or int64" in lib.fsc_last_error()
    assert lib.fsc_adamw_values(-1, 0, None, None, None, None) == 1
    assert lib.fsc_adamw_step(-1, None, None, None, None) == 1


def test_grid_of_the_8_bit_states():
    for root, n, fraction in ((False, 128, 3), (True, 256, 4)):
        g = O.grid(root)
        assert len(g) == n and g[-1] == 1.0 and g[0] == 0.0 and (np.diff(g) > 0).all()
        assert np.array_equal(g, g.astype(np.float32))
        # neighbours are a share 2^-fraction or less apart
        assert (np.diff(g[1:]) / g[1:-1]).max() == 2.0 ** -fraction


def test_8_bit_rounding_keeps_the_mean():
    """Over many steps (other random numbers) the mean of what a value is rounded to is the value: 4,000 roundings of a
    step s scatter by at most s / 2 each, their mean by s / 2 / sqrt(4000), and six of those are not passed."""
    rng = np.random.default_rng(5)
    for root in (False, True):
        x = np.exp(rng.uniform(-8, 0, 256)).astype(np.float32)
        x[0] = 1.0
        total = np.zeros(256)
        for step in range(4000):
            total += O.decode(*O.encode(x, step, root), root)
        spread = x * 2.0 ** -(4 if root else 3) / 2 / np.sqrt(4000)
        assert (np.abs(total / 4000 - x) <= 6 * spread + 1e-7 * x).all()


@pytest.mark.parametrize("shape", [(2 ** 20 + 1,), (2 ** 31 + 5,), (2 ** 32 + 8,)])
def test_lookups_of_wider_rows_are_refused(shape):
    """Also where the width's lower 32 bits by themselves are a width."""
    with pytest.raises(RuntimeError, match="at most 2\\^20"):
        L.embedding(meta(1, *shape), meta(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="at most 2\\^20"):
        torch.ops.fsctep.embedding_backward(meta(3, *shape), meta(3, dtype=torch.int64), 2, 1.0)


def test_step_of_a_trunk_checks_what_it_is_compared_with():
    """A column of energies would be compared with every structure's, one row of forces with every atom's."""
    class Trunk(torch.nn.Module):
        def forward_graph(self, *args, **kwargs):
            raise AssertionError("run before the check")

    pos, batch, cell, e = torch.zeros(5, 3), torch.zeros(5, dtype=torch.int64), torch.zeros(2, 3, 3), torch.zeros(2)
    w = torch.zeros(3, requires_grad=True)
    opt = optim.AdamW([w])
    for energy, forces in ((e[:, None], pos), (e[:1], pos), (e[0], pos), (e, pos[:1]), (e, pos.t()), (e, pos[0])):
        with pytest.raises(ValueError, match="energy must be"):
            optim.train_step(Trunk().train(), opt, pos, batch, cell, None, energy, forces)


@pytest.mark.parametrize("variant", ["amsgrad", "maximize"])
def test_checkpoints_of_other_optimisers_are_refused(variant):
    p, q = torch.zeros(3, requires_grad=True), torch.zeros(3, requires_grad=True)
    theirs, mine = torch.optim.AdamW([p], lr=0.5, **{variant: True}), optim.AdamW([q], lr=0.25)
    p.grad = torch.ones(3)
    theirs.step()
    with pytest.raises(ValueError, match=variant):
        mine.load_state_dict(theirs.state_dict())
    assert mine.param_groups[0]["lr"] == 0.25 and not mine.state


def test_checkpoints_of_other_states_leave_the_optimiser_as_it_was():
    p, q = torch.zeros(300, requires_grad=True), torch.zeros(300, requires_grad=True)
    theirs, mine = torch.optim.AdamW([p], lr=0.5), optim.AdamW([q], lr=0.25, state_bits=8)
    p.grad = torch.ones(300)
    theirs.step()
    with pytest.raises(ValueError, match="8 bits"):
        mine.load_state_dict(theirs.state_dict())
    assert mine.param_groups[0]["lr"] == 0.25 and not mine.state


def test_step_of_a_trunk_is_not_captured(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    pos, batch, cell = torch.zeros(5, 3), torch.zeros(5, dtype=torch.int64), torch.zeros(2, 3, 3)
    opt = optim.AdamW([torch.zeros(3, requires_grad=True)])
    with pytest.raises(RuntimeError, match="captured"):
        optim.train_step(torch.nn.Linear(2, 2), opt, pos, batch, cell, None, torch.zeros(2), pos)
