"""The experts' products through the C ABI with every output and workspace of the size that is asked for inside a larger
buffer whose bytes around it have to stay; values against the 64-bit oracle within the bounds of test_experts_gpu.py (fp32
1e-5, bf16 2^-7 of the largest value)."""

import ctypes

import pytest
import torch

from oracle import experts as O
from test_experts_gpu import DEV, DT, HANDFUL, MLP, NORM, ROUTE, TILES, TOL, close, problem
from test_experts_host import Dims

pytestmark = pytest.mark.gpu
GUARD = 8 << 20            # bytes on each side: more than any expert's matrices here
FILL = 0xA5


class Guarded:
    """`shape` values of a type between guard bytes."""

    def __init__(self, shape, dtype):
        self.n = torch.empty(0, dtype=dtype).element_size() * int(torch.Size(shape).numel())
        self.buf = torch.full((2 * GUARD + self.n,), FILL, dtype=torch.uint8, device=DEV)
        self.t = self.buf[GUARD:GUARD + self.n].view(dtype).view(shape)

    @property
    def ptr(self):
        return self.buf.data_ptr() + GUARD

    def check(self, what):
        assert int((self.buf[:GUARD] != FILL).sum()) == 0, f"{what}: bytes before"
        assert int((self.buf[GUARD + self.n:] != FILL).sum()) == 0, f"{what}: bytes after"


def run(x, index, weight, w_in, w_out, dy):
    """(y, dx, dweight, dw_in, dw_out) of rows x, dy with their own strides; guards checked."""
    from fsctep_amd import _lib
    rows, width = x.shape
    E, hidden, k = w_out.shape[0], w_out.shape[2], index.shape[1]
    d = Dims(rows, width, hidden, E, k, 0 if x.dtype == torch.float32 else 1)
    n = [ctypes.c_int64() for _ in range(4)]
    _lib.call("fsc_expert_sizes", ctypes.byref(d), *(ctypes.byref(v) for v in n))
    plan, saved, fwd, bwd = (v.value for v in n)
    g = dict(plan=Guarded((plan,), torch.int32), saved=Guarded((saved,), torch.float32), forward=Guarded((fwd,), torch.uint8),
             backward=Guarded((bwd,), torch.uint8), y=Guarded(x.shape, x.dtype), dx=Guarded(x.shape, x.dtype),
             dweight=Guarded(weight.shape, torch.float32), dw_in=Guarded(w_in.shape, x.dtype),
             dw_out=Guarded(w_out.shape, x.dtype))
    p, st = {name: b.ptr for name, b in g.items()}, _lib.stream_handle(DEV)
    _lib.call("fsc_expert_plan", ctypes.byref(d), index.data_ptr(), p["plan"], st)
    _lib.call("fsc_expert_mlp_forward", ctypes.byref(d), x.stride(0), x.data_ptr(), index.data_ptr(), p["plan"],
              weight.data_ptr(), w_in.data_ptr(), w_out.data_ptr(), p["saved"], p["forward"], p["y"], st)
    _lib.call("fsc_expert_mlp_backward", ctypes.byref(d), x.stride(0), dy.stride(0), dy.data_ptr(), x.data_ptr(),
              index.data_ptr(), p["plan"], weight.data_ptr(), w_in.data_ptr(), w_out.data_ptr(), p["saved"], p["backward"],
              p["dx"], p["dweight"], p["dw_in"], p["dw_out"], st)
    torch.cuda.synchronize()
    for name, b in g.items():
        b.check(name)
    return [g[name].t for name in ("y", "dx", "dweight", "dw_in", "dw_out")]


def reference(x, index, weight, w_in, w_out, dy):
    leaf = [t.double().requires_grad_(True) for t in (x, weight, w_in, w_out)]
    y = O.expert_mlp(leaf[0], index, leaf[1], leaf[2], leaf[3])
    return [y.detach(), *torch.autograd.grad(y, leaf, dy.double())]


# Slots as many as the share of a weight gradient, one fewer and one more: of both gradients (fp32 128, bf16 256 and, few
# for each expert, 128) or of dw_in alone (1,024 and 2,048).
SHARES = [("fp32", 64, 640, 640, 2, 2), ("fp32", 64, 640, 640, 3, 2), ("fp32", 127, 330, 203, 2, 1), ("fp32", 128, 330, 203, 2, 1),
          ("fp32", 129, 330, 203, 2, 1), ("fp32", 512, 640, 640, 16, 2), ("bf16", 64, 640, 640, 8, 2),
          ("bf16", 128, 640, 640, 4, 2), ("bf16", 255, 200, 72, 3, 1), ("bf16", 256, 200, 72, 3, 1), ("bf16", 257, 200, 72, 3, 1),
          ("bf16", 1024, 640, 640, 16, 2)]


@pytest.mark.parametrize("dtype,rows,width,hidden,experts,k", SHARES)
def test_weight_gradients_stay_inside_their_arrays(dtype, rows, width, hidden, experts, k):
    p = problem(rows, width, hidden, experts, k, DT[dtype], rows + experts)
    got = run(*(t.to(DEV) for t in p))
    for a, b, n in zip(got, reference(*p), ("y", "dx", "dweight", "dw_in", "dw_out")):
        close(a, b, TOL[DT[dtype]], n)


def held_rows(hold, t, stride, at):
    """Rows t as a view of `hold` (uint8) with a row stride in elements, from element `at` on."""
    v = hold.view(t.dtype).as_strided(t.shape, (stride, 1), at)
    v.copy_(t)
    return v


# Row strides that put the last rows past what a buffer of 32-bit offsets reaches (0xF0000000 bytes), rows by tiles and few;
# and rows at odd places, whole words or not, which are copied.
@pytest.mark.parametrize("rows,width,far", [(300, 64, True), (40, 64, True), (300, 65, True), (300, 64, False), (300, 65, False)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_strided_rows_stay_inside_the_workspaces(rows, width, far, dtype):
    dt = DT[dtype]
    size = 4 if dtype == "fp32" else 2
    x, index, weight, w_in, w_out, dy = problem(rows, width, 40, 4, 2, dt, rows + width)
    stride = (0xF0000000 // (rows - 1) // size + 4) // 4 * 4 + 4 if far else 203
    hold = torch.empty(rows * stride * size + 1024, dtype=torch.uint8, device=DEV)
    xs, dys = held_rows(hold, x.to(DEV), stride, 1), held_rows(hold, dy.to(DEV), stride, 101)
    got = run(xs, index.to(DEV), weight.to(DEV), w_in.to(DEV), w_out.to(DEV), dys)
    for a, b, n in zip(got, reference(x, index, weight, w_in, w_out, dy), ("y", "dx", "dweight", "dw_in", "dw_out")):
        close(a, b, TOL[dt], n)


@pytest.mark.parametrize("rows,width,hidden", [(300, 65, 41), (300, 64, 40), (20, 65, 41), (2, 65, 41)])
def test_8_bit_products_stay_inside_the_workspaces(rows, width, hidden):
    from fsctep_amd import _lib, expert_ops as X
    x, index, weight, w_in, w_out, _ = problem(rows, width, hidden, 4, 2, torch.float32, rows + width)
    (q, s), (qi, si), (qo, so) = X.to_codes(x.to(DEV)), X.to_codes(w_in.to(DEV)), X.to_codes(w_out.to(DEV))
    hold = torch.zeros(rows * 203 + 1024, dtype=torch.uint8, device=DEV)
    v = held_rows(hold, q, 203, 3)
    d = Dims(rows, width, hidden, 4, 2, 2)
    n = [ctypes.c_int64() for _ in range(4)]
    _lib.call("fsc_expert_sizes", ctypes.byref(d), *(ctypes.byref(t) for t in n))
    plan, ws = Guarded((n[0].value,), torch.int32), Guarded((n[2].value,), torch.uint8)
    y, st = Guarded(x.shape, torch.bfloat16), _lib.stream_handle(DEV)
    i, w = index.to(DEV), weight.to(DEV)
    _lib.call("fsc_expert_plan", ctypes.byref(d), i.data_ptr(), plan.ptr, st)
    _lib.call("fsc_expert_mlp_q8", ctypes.byref(d), 203, v.data_ptr(), s.data_ptr(), i.data_ptr(), plan.ptr, w.data_ptr(),
              qi.data_ptr(), si.data_ptr(), qo.data_ptr(), so.data_ptr(), ws.ptr, y.ptr, st)
    torch.cuda.synchronize()
    for b, name in ((plan, "plan"), (ws, "workspace"), (y, "y")):
        b.check(name)
    assert torch.equal(y.t, X.expert_mlp_q8(q, s, i, w, qi, si, qo, so))


@pytest.mark.parametrize("rows,width,hidden,experts,k", MLP + TILES + HANDFUL)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_products_stay_inside_their_arrays(rows, width, hidden, experts, k, dtype):
    p = problem(rows, width, hidden, experts, k, DT[dtype], rows + width)
    got = run(*(t.to(DEV) for t in p))
    for a, b, n in zip(got, reference(*p), ("y", "dx", "dweight", "dw_in", "dw_out")):
        close(a, b, TOL[DT[dtype]], n)


@pytest.mark.parametrize("rows,width", NORM)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_stays_inside_its_arrays(rows, width, dtype, residual):
    from fsctep_amd import _lib
    dt, code = DT[dtype], 0 if dtype == "fp32" else 1
    x, r, dy, dz = (torch.randn(rows, width + 3, device=DEV).to(dt)[:, 1:width + 1] for _ in range(4))
    w, eps, st = torch.randn(width, device=DEV).to(dt), 1e-6, _lib.stream_handle(DEV)
    n = ctypes.c_int64()
    _lib.call("fsc_rms_norm_workspace", rows, width, ctypes.byref(n))
    like = lambda t=dt, shape=(rows, width): Guarded(shape, t)
    g = dict(y=like(), z=like(), rstd=like(torch.float32, (rows,)), codes=like(torch.int8), scale=like(torch.float32, (rows,)),
             z8=like(), dx=like(), dw=like(dt, (width,)), workspace=like(torch.float32, (n.value,)))
    rp, zp = (r.data_ptr(), g["z"].ptr) if residual else (0, 0)
    s = width + 3
    _lib.call("fsc_rms_norm_forward", rows, width, code, code, s, s, x.data_ptr(), rp, w.data_ptr(), eps, g["y"].ptr, zp,
              g["rstd"].ptr, st)
    _lib.call("fsc_rms_norm_q8", rows, width, code, code, s, s, x.data_ptr(), rp, w.data_ptr(), eps, g["codes"].ptr,
              g["scale"].ptr, g["z8"].ptr if residual else 0, st)
    z, zs = (g["z"].ptr, width) if residual else (x.data_ptr(), s)
    _lib.call("fsc_rms_norm_backward", rows, width, code, code, zs, s, s, z, w.data_ptr(), g["rstd"].ptr, eps, dy.data_ptr(),
              dz.data_ptr() if residual else 0, g["dx"].ptr, g["dw"].ptr, g["workspace"].ptr, st)
    torch.cuda.synchronize()
    for name, b in g.items():
        b.check(name)
    leaf = [t.cpu().double().requires_grad_(True) for t in (x, w, r)]
    y0, z0 = O.rms_norm(leaf[0], leaf[1], leaf[2] if residual else None, held=dt)
    heads, gs = ((y0, z0), (dy, dz)) if residual else ((y0,), (dy,))
    dx0, dw0 = torch.autograd.grad(heads, leaf[:2], [t.cpu().double() for t in gs])
    for a, b, name in ((g["y"], y0, "y"), (g["dx"], dx0, "dx"), (g["dw"], dw0, "dw")):
        close(a.t, b, TOL[dt], name)


@pytest.mark.parametrize("rows,experts,k,groups,kept,best", ROUTE)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_router_stays_inside_its_arrays(rows, experts, k, groups, kept, best, dtype):
    from fsctep_amd import _lib, expert_ops as X
    dt, code, st = DT[dtype], 0 if dtype == "fp32" else 1, _lib.stream_handle(DEV)
    l = torch.randn(rows, experts + 5, device=DEV).to(dt)[:, 2:experts + 2]
    bias = 0.1 * torch.randn(experts, device=DEV)
    u = torch.randn(rows, k, device=DEV)
    for score, name in ((0, "softmax"), (1, "sigmoid")):
        for renormalise in (0, 1):
            g = dict(index=Guarded((rows, k), torch.int32), weight=Guarded((rows, k), torch.float32), dl=Guarded((rows, experts), dt))
            _lib.call("fsc_route_experts", rows, experts, code, experts + 5, l.data_ptr(), bias.data_ptr(), k, score, groups, kept,
                      best, renormalise, 1.5, g["index"].ptr, g["weight"].ptr, st)
            _lib.call("fsc_route_experts_backward", rows, experts, code, experts + 5, l.data_ptr(), g["index"].ptr,
                      g["weight"].ptr, u.data_ptr(), k, score, renormalise, 1.5, g["dl"].ptr, st)
            torch.cuda.synchronize()
            for what, b in g.items():
                b.check(what)
            i, w = X.route_experts(l, k, score=name, bias=bias, groups=groups, groups_kept=kept, group_best=best,
                                   renormalise=bool(renormalise), scale=1.5)
            assert torch.equal(i, g["index"].t) and torch.equal(w, g["weight"].t)
            want = O.route_gradient(l.cpu().double(), i.cpu(), name, bool(renormalise), 1.5, u.cpu().double())
            close(g["dl"].t, want, 2e-5 if dtype == "fp32" else TOL[dt], "dlogits")
