"""GPU parity of the expert readout's operators against the 64-bit oracle (oracle/experts.py) on the same inputs.

Bounds, set from the arithmetic.  fp32 paths: sums of at most 2,600 products with 24-bit operands and 32-bit
accumulators, relative error of a result's norm within a few 2^-24 sqrt(K); 1e-5 of the largest value (the bound
of the framework's other fp32 operators).  bf16 paths: operands exact, at most one rounding of a held value and
one of the output, each 2^-9: 2^-7 of the largest value.  8-bit products: whole numbers are exact; a hidden value
next to a half code may take either neighbour (1/127 of its group's largest) and the output is rounded to bf16:
2^-6.  Codes, indices and repeated runs: equal.
"""

import math

import pytest
import torch

from oracle import experts as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOL = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -7}
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


def X():
    from fsctep_amd import expert_ops
    return expert_ops


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def rn(g, *shape):
    return torch.randn(*shape, generator=g, dtype=torch.float64)


def close(got, ref, tol, what=""):
    got, ref = got.detach().double().cpu(), ref.detach().double().cpu()
    assert got.shape == ref.shape, what
    if ref.numel() == 0:
        return
    err, top = float((got - ref).abs().max()), float(ref.abs().max())
    assert err <= tol * max(top, 1e-30), (what, err, top)


# ------------------------------------------------------------------ norm
NORM = [(1, 1), (1, 640), (3, 7), (33, 640), (5, 130), (257, 1600), (64, 331), (7, 2048), (2, 5000), (9, 515), (3, 2052)]


@pytest.mark.parametrize("rows,width", NORM)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_and_gradients(rows, width, dtype, residual):
    dt, g = DT[dtype], gen(rows * 7 + width)
    size = torch.exp(rn(g, rows, 1))
    x, r = (size * rn(g, rows, width)).to(dt), (size * rn(g, rows, width)).to(dt)
    w, dy, dz = (1 + 0.3 * rn(g, width)).to(dt), rn(g, rows, width).to(dt), rn(g, rows, width).to(dt)
    leaf = [t.double().requires_grad_(True) for t in (x, w, r)]
    y0, z0 = O.rms_norm(leaf[0], leaf[1], leaf[2] if residual else None, held=dt)
    heads, gs = ((y0, z0), (dy.double(), dz.double())) if residual else ((y0,), (dy.double(),))
    ref = torch.autograd.grad(heads, leaf[:3 if residual else 2], gs)
    dev = [t.to(DEV).requires_grad_(True) for t in (x, w, r)]
    y, z = X().rms_norm(dev[0], dev[1], dev[2] if residual else None)
    heads, gs = ((y, z), (dy.to(DEV), dz.to(DEV))) if residual else ((y,), (dy.to(DEV),))
    got = torch.autograd.grad(heads, dev[:3 if residual else 2], gs)
    close(y, y0, TOL[dt], "y")
    assert torch.equal(z.detach().cpu(), z0.detach().to(dt))
    for a, b, n in zip(got, ref, ("dx", "dw", "dr")):
        close(a, b, TOL[dt], n)


@pytest.mark.parametrize("rows,width", [(1, 640), (37, 640), (5, 331), (2, 5000), (11, 129)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_norm_codes(rows, width, dtype):
    """The codes of the 32-bit y, its root rounded from a 64-bit sum: equal, whatever the order of the sum."""
    dt, g = DT[dtype], gen(rows + width)
    x, r = rn(g, rows, width).to(dt), rn(g, rows, width).to(dt)
    w = (1 + 0.3 * rn(g, width)).to(torch.float32)
    x[0] = 0
    r[0] = 0
    q, s, z = X().rms_norm_q8(x.to(DEV), w.to(DEV), r.to(DEV))
    zc = (x.float() + r.float()).to(dt).float()
    assert torch.equal(z.cpu().float(), zc)
    rstd = (1 / torch.sqrt((zc.double() ** 2).mean(1, keepdim=True) + 1e-6)).float()
    y = zc * rstd * w
    top = y.abs().amax(1, keepdim=True)
    code = torch.where(top > 0, torch.round(y * torch.div(torch.full_like(top, 127.0), top)), torch.zeros_like(y))
    assert torch.equal(q.cpu().float(), code)
    assert torch.equal(s.cpu(), (top / 127).squeeze(1))
    assert int(q[0].abs().max()) == 0 and float(s[0]) == 0


def test_norm_mixed_weight_strides_and_alignment():
    """A float32 weight with bfloat16 rows; rows that are slices (row stride above the width, odd offsets)."""
    g = gen(3)
    for dt, off, width in ((torch.float32, 0, 640), (torch.float32, 3, 641), (torch.bfloat16, 8, 640), (torch.bfloat16, 5, 333)):
        big, w = rn(g, 19, 1400).to(dt), (1 + 0.3 * rn(g, width)).float()
        x, r = big[:, off:off + width], big[:, 700 + off:700 + off + width] if off + 700 + width <= 1400 else big[:, :width]
        y0, z0 = O.rms_norm(x, w, r, held=dt)
        bd = big.to(DEV)
        xd = bd[:, off:off + width]
        rd = bd[:, 700 + off:700 + off + width] if off + 700 + width <= 1400 else bd[:, :width]
        y, z = X().rms_norm(xd, w.to(DEV) if dt == torch.bfloat16 else w.to(dt).to(DEV), rd)
        close(y, y0, TOL[dt])
        close(z, z0, TOL[dt])


def test_norm_special_rows():
    x = torch.ones(5, 640, device=DEV)
    x[0, 3], x[1, 5], x[2] = float("nan"), float("inf"), 0
    w = torch.ones(640, device=DEV)
    y, _ = X().rms_norm(x, w)
    assert torch.isnan(y[0]).all() and torch.isnan(y[1, 5]) and float(y[1, :5].abs().max()) == 0
    assert float(y[2].abs().max()) == 0 and torch.isfinite(y[3:]).all()
    q, s, _ = X().rms_norm_q8(x, w)
    assert torch.isnan(s[0]) and torch.isnan(s[1]) and torch.isfinite(s[2:]).all() and int(q[0].abs().max()) == 0
    y, z = X().rms_norm(torch.empty(0, 640, device=DEV), w)
    assert y.shape == (0, 640)
    xe = torch.empty(0, 640, device=DEV, requires_grad=True)
    we = torch.ones(640, device=DEV, requires_grad=True)
    y, _ = X().rms_norm(xe, we)
    dx, dw = torch.autograd.grad(y, (xe, we), torch.empty(0, 640, device=DEV))
    assert dx.shape == (0, 640) and float(dw.abs().max()) == 0


# ------------------------------------------------------------------ router
ROUTE = [(1, 8, 2, 1, 1, 1), (33, 8, 2, 1, 1, 1), (5, 1, 1, 1, 1, 1), (40, 5, 5, 1, 1, 1), (17, 160, 6, 8, 3, 2),
         (9, 256, 8, 8, 4, 2), (21, 64, 4, 4, 1, 1), (3, 512, 16, 1, 1, 1), (50, 33, 3, 3, 2, 2), (8, 24, 4, 8, 2, 1),
         (6, 256, 3, 128, 2, 2)]


@pytest.mark.parametrize("rows,experts,k,groups,kept,best", ROUTE)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("renormalise", [False, True])
def test_route(rows, experts, k, groups, kept, best, score, bias, renormalise):
    g = gen(rows * experts + k)
    # logits on a grid, so that equal scores are exact ties and different ones stay apart in 32 bits
    logits = (torch.round(8 * rn(g, rows, experts)) / 8).float()
    logits[torch.rand(rows, experts, generator=g) < 0.1] = -math.inf
    if rows > 2:
        logits[1] = -math.inf                      # a row with nothing to choose
        logits[2] = 0.0                            # a row of ties
    b = (torch.round(16 * rn(g, experts)) / 64).float() if bias else None
    s = O.scores(logits, score).float()            # 32-bit scores: equal ones tie
    c = s if b is None else s + b
    c = torch.where(logits > -math.inf, c, torch.full_like(c, -math.inf))
    u = rn(g, rows, k).float()
    ld = logits.to(DEV).requires_grad_(True)
    index, weight = X().route_experts(ld, k, score=score, bias=None if b is None else b.to(DEV), groups=groups,
                                      groups_kept=kept, group_best=best, renormalise=renormalise, scale=1.5)
    dl, = torch.autograd.grad(weight, ld, u.to(DEV))
    got = index.cpu()
    # the choice: c of the chosen, in order, is that of the oracle's choice to the last bits of 32, and where the
    # oracle's neighbours differ by more than that the experts are the same
    ref = O.choose(c.double(), k, groups, kept, best)
    pick = lambda i: torch.where(i >= 0, c.gather(1, i.clamp(min=0).long()), torch.full_like(weight.cpu(), -math.inf))
    assert torch.equal(ref < 0, got < 0)
    same = torch.where(got >= 0, (pick(ref) - pick(got)).abs() <= 4e-7, torch.ones_like(got, dtype=torch.bool))
    if groups == 1:
        assert same.all()
        if b is None:
            assert torch.equal(ref, got)           # monotone scores: the order is that of the logits
    else:
        assert (ref == got).all(1).float().mean() > 0.9
    w0 = O.weights(logits.double(), got, score, renormalise, 1.5)
    close(weight, w0, 1e-5, "weight")
    close(dl, O.route_gradient(logits.double(), got, score, renormalise, 1.5, u.double()), 2e-5, "dlogits")


def test_route_gradient_against_differences():
    g = gen(11)
    l = rn(g, 6, 12).float()
    u = rn(g, 6, 3)
    for score in ("softmax", "sigmoid"):
        for renorm in (False, True):
            ld = l.to(DEV).requires_grad_(True)
            index, w = X().route_experts(ld, 3, score=score, renormalise=renorm)
            dl, = torch.autograd.grad(w, ld, u.float().to(DEV))
            for t, e in ((0, int(index[0, 1])), (3, 5), (5, int(index[5, 2]))):
                h = 1e-5
                d = []
                for sgn in (1, -1):
                    p = l.double().clone()
                    p[t, e] += sgn * h
                    d.append(float((O.weights(p, index.cpu(), score, renorm) * u).sum()))
                assert abs((d[0] - d[1]) / (2 * h) - float(dl[t, e])) < 1e-5


def test_route_bf16_strides_ties_and_nan():
    l = torch.zeros(4, 40, device=DEV, dtype=torch.bfloat16)
    view = l[:, 3:23]                              # an odd offset, a row stride above the row
    index, w = X().route_experts(view, 4)
    assert torch.equal(index.cpu(), torch.arange(4).int().expand(4, 4)) and torch.allclose(w, torch.full_like(w, 0.25))
    big = torch.full((3, 8), -3.0e38, device=DEV)  # the type's lowest values are still choosable
    index, w = X().route_experts(big, 2)
    assert torch.equal(index.cpu(), torch.tensor([[0, 1]] * 3).int()) and torch.allclose(w, torch.full_like(w, 0.5))
    bad = torch.randn(3, 8, device=DEV)
    bad[1, 4] = float("nan")
    index, w = X().route_experts(bad, 2, score="sigmoid")
    assert torch.isnan(w[1]).all() and index[1].tolist() == [0, 1] and torch.isfinite(w[[0, 2]]).all()
    under = torch.full((2, 8), -200.0, device=DEV)  # sigmoids that are 0 in 32 bits: nothing to renormalise by
    index, w = X().route_experts(under, 2, score="sigmoid")
    assert float(w.abs().max()) == 0 and int(index.min()) == 0
    index, w = X().route_experts(torch.empty(0, 8, device=DEV), 2)
    assert index.shape == (0, 2) and w.shape == (0, 2)


# ------------------------------------------------------------------ products
def problem(rows, width, hidden, experts, k, dt, seed, empty=True):
    g = gen(seed)
    x = rn(g, rows, width).to(dt)
    w_in, w_out = (rn(g, experts, 2 * hidden, width) / math.sqrt(width)).to(dt), (rn(g, experts, width, hidden) / math.sqrt(hidden)).to(dt)
    index = torch.rand(rows, experts, generator=g).argsort(1)[:, :k].int()
    if empty and rows > 2:
        index[rows // 2] = -1                       # a row with no expert
        index[0, -1] = experts + 3                  # an index outside
        index[index == experts - 1] = 0 if k == 1 else -1   # an expert that nobody chose
    weight = torch.rand(rows, k, generator=g) + 0.1
    return x, index.contiguous(), weight, w_in, w_out, rn(g, rows, width).to(dt)


# rows, width, hidden, experts, k: single rows, sizes around every tile, primes, many experts, all rows on one expert
MLP = [(1, 640, 640, 8, 2), (1, 7, 5, 3, 1), (2, 64, 64, 2, 2), (15, 33, 17, 4, 3), (16, 128, 64, 1, 1), (17, 96, 130, 3, 2),
       (33, 640, 320, 8, 2), (100, 331, 203, 5, 2), (129, 130, 66, 2, 1), (300, 72, 136, 3, 2), (700, 264, 128, 4, 2),
       (64, 48, 40, 64, 4), (1000, 40, 24, 1, 1), (2500, 24, 16, 7, 4),
       (4100, 16, 8, 300, 3), (513, 36, 1, 2, 1), (40, 1, 9, 2, 1)]


@pytest.mark.parametrize("rows,width,hidden,experts,k", MLP)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_products_and_gradients(rows, width, hidden, experts, k, dtype):
    dt = DT[dtype]
    x, index, weight, w_in, w_out, dy = problem(rows, width, hidden, experts, k, dt, rows + width)
    leaf = [t.double().requires_grad_(True) for t in (x, weight, w_in, w_out)]
    y0 = O.expert_mlp(leaf[0], index, leaf[1], leaf[2], leaf[3])
    ref = torch.autograd.grad(y0, leaf, dy.double())
    dev = [t.to(DEV).requires_grad_(True) for t in (x, weight, w_in, w_out)]
    with torch.no_grad():
        plain = X().expert_mlp(dev[0], index.to(DEV), dev[1], dev[2], dev[3])
    y = X().expert_mlp(dev[0], index.to(DEV), dev[1], dev[2], dev[3])
    got = torch.autograd.grad(y, dev, dy.to(DEV), retain_graph=True)
    only, = torch.autograd.grad(y, dev[0], dy.to(DEV))
    assert torch.equal(plain, y) and torch.equal(only, got[0])
    close(y, y0, TOL[dt], "y")
    for a, b, n in zip(got, ref, ("dx", "dweight", "dw_in", "dw_out")):
        assert a.dtype == (torch.float32 if n == "dweight" else dt)
        close(a, b, TOL[dt], n)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_products_repeat_to_the_bit(dtype):
    dt = DT[dtype]
    x, index, weight, w_in, w_out, dy = (t.to(DEV) for t in problem(700, 200, 136, 5, 2, dt, 4))
    outs = []
    for _ in range(2):
        leaf = [t.clone().requires_grad_(True) for t in (x, weight, w_in, w_out)]
        y = X().expert_mlp(leaf[0], index, leaf[1], leaf[2], leaf[3])
        outs.append((y, *torch.autograd.grad(y, leaf, dy)))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_products_gradient_against_differences():
    x, index, weight, w_in, w_out, dy = problem(6, 20, 12, 3, 2, torch.float32, 9, empty=False)
    dev = [t.to(DEV).requires_grad_(True) for t in (x, weight, w_in, w_out)]
    y = X().expert_mlp(dev[0], index.to(DEV), dev[1], dev[2], dev[3])
    got = torch.autograd.grad(y, dev, dy.to(DEV))
    e = int(index[2, 1])
    for which, at in ((0, (2, 5)), (1, (2, 1)), (2, (e, 3, 7)), (2, (e, 15, 7)), (3, (e, 4, 2))):
        d, h = [], 1e-5
        for sgn in (1, -1):
            p = [t.double().clone() for t in (x, weight, w_in, w_out)]
            p[which][at] += sgn * h
            d.append(float((O.expert_mlp(p[0], index, p[1], p[2], p[3]) * dy.double()).sum()))
        assert abs((d[0] - d[1]) / (2 * h) - float(got[which][at])) < 1e-4 * max(1.0, abs(d[0] - d[1]) / (2 * h))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_products_strides_and_expanded_gradient(dtype):
    """Rows that are slices with odd offsets, a transposed gradient and one expanded from a scalar."""
    dt = DT[dtype]
    x, index, weight, w_in, w_out, dy = problem(70, 64, 40, 4, 2, dt, 21)
    y0 = O.expert_mlp(x, index, weight, w_in, w_out)
    pad = torch.full((70, 200), float("nan"), dtype=dt, device=DEV)
    for off in (8, 3):
        v = pad[:, off:off + 64]
        v.copy_(x)
        close(X().expert_mlp(v, index.to(DEV), weight.to(DEV), w_in.to(DEV), w_out.to(DEV)), y0, TOL[dt])
    leaf = x.double().requires_grad_(True)
    ref, = torch.autograd.grad(O.expert_mlp(leaf, index, weight, w_in, w_out).sum(), leaf)
    xd = x.to(DEV).requires_grad_(True)
    y = X().expert_mlp(xd, index.to(DEV), weight.to(DEV), w_in.to(DEV), w_out.to(DEV))
    close(torch.autograd.grad(y.sum(), xd)[0], ref, TOL[dt])


def test_products_keep_rows_apart():
    """A NaN or an infinity in one row, or in an expert nobody chose, stays there."""
    x, index, weight, w_in, w_out, dy = problem(150, 64, 40, 4, 2, torch.float32, 5)
    y0 = O.expert_mlp(x, index, weight, w_in, w_out)
    x[7, 3], x[90, 1] = float("nan"), float("inf")
    w_in[3], w_out[3] = float("nan"), float("inf")      # expert 3 is the one that nobody chose
    y = X().expert_mlp(x.to(DEV), index.to(DEV), weight.to(DEV), w_in.to(DEV), w_out.to(DEV)).cpu()
    ok = torch.ones(150, dtype=torch.bool)
    ok[[7, 90]] = False
    close(y[ok], y0[ok], 1e-5)
    if bool((index[7] >= 0).any() & (index[7] < 4).any()):
        assert not torch.isfinite(y[7]).any()


def test_products_of_very_different_sizes():
    """Rows and experts across 60 powers of two: each is as accurate as alone (no shared scale)."""
    x, index, weight, w_in, w_out, _ = problem(64, 96, 64, 3, 1, torch.float32, 8, empty=False)
    x = x * torch.exp2(torch.linspace(-30, 10, 64)).unsqueeze(1)
    y0 = O.expert_mlp(x, index, weight, w_in, w_out)
    y = X().expert_mlp(x.to(DEV), index.to(DEV), weight.to(DEV), w_in.to(DEV), w_out.to(DEV)).double().cpu()
    err = (y - y0).abs().amax(1) / y0.abs().amax(1)
    assert float(err.max()) < 1e-5


def test_products_empty():
    for dt in (torch.float32, torch.bfloat16):
        x = torch.empty(0, 64, device=DEV, dtype=dt, requires_grad=True)
        idx, w = torch.empty(0, 2, device=DEV, dtype=torch.int32), torch.empty(0, 2, device=DEV)
        w_in = torch.randn(3, 80, 64, device=DEV).to(dt).requires_grad_(True)
        w_out = torch.randn(3, 64, 40, device=DEV).to(dt).requires_grad_(True)
        y = X().expert_mlp(x, idx, w, w_in, w_out)
        assert y.shape == (0, 64)
        for t in torch.autograd.grad(y, (x, w_in, w_out), torch.empty(0, 64, device=DEV, dtype=dt)):
            assert t.numel() == 0 or float(t.abs().max()) == 0
        x1 = torch.randn(9, 64, device=DEV).to(dt).requires_grad_(True)
        none = torch.full((9, 2), -1, device=DEV, dtype=torch.int32)
        y = X().expert_mlp(x1, none, torch.ones(9, 2, device=DEV), w_in, w_out)
        grads = torch.autograd.grad(y, (x1, w_in, w_out), torch.ones_like(y))
        assert float(y.abs().max()) == 0 and all(float(t.abs().max()) == 0 for t in grads)


Q8 = [(1, 640, 640, 8, 2), (33, 640, 320, 8, 2), (5, 17, 40, 2, 1), (100, 331, 203, 5, 2), (300, 128, 256, 3, 2),
      (700, 64, 130, 4, 1), (40, 16, 128, 64, 4), (3000, 32, 48, 5, 3)]


@pytest.mark.parametrize("rows,width,hidden,experts,k", Q8)
def test_products_in_8_bits(rows, width, hidden, experts, k):
    x, index, weight, w_in, w_out, _ = problem(rows, width, hidden, experts, k, torch.float32, rows + hidden)
    (q, s), (qi, si), (qo, so) = X().to_codes(x.to(DEV)), X().to_codes(w_in.to(DEV)), X().to_codes(w_out.to(DEV))
    y = X().expert_mlp_q8(q, s, index.to(DEV), weight.to(DEV), qi, si, qo, so)
    full = lambda c, u: c.cpu().double() * u.cpu().double().unsqueeze(-1)
    y0 = O.expert_mlp(full(q, s), index, weight, full(qi, si), full(qo, so), group=128)
    assert y.dtype == torch.bfloat16
    close(y, y0, 2.0 ** -6)
    # and near the products of the values before the codes: 8-bit rows, weights and hidden values
    near = O.expert_mlp(x, index, weight, w_in, w_out)
    assert float((y.cpu().double() - near).norm() / near.norm()) < 0.05


# ------------------------------------------------------------------ streams, graphs, devices of use
def test_operators_on_a_side_stream_and_in_a_graph():
    x, index, weight, w_in, w_out, _ = (t.to(DEV) for t in problem(50, 64, 40, 4, 2, torch.float32, 2))
    norm, gate = torch.ones(64, device=DEV), torch.randn(4, 64, device=DEV)

    def block(v):
        y, _ = X().rms_norm(v, norm)
        i, w = X().route_experts((y.unsqueeze(1) * gate).sum(-1), 2)
        return v + X().expert_mlp(y, i, w, w_in, w_out)

    want = block(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = block(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, other)
    static = x.clone()
    with torch.cuda.stream(side):
        block(static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(static)
    for seed in range(4):
        v = torch.randn(50, 64, device=DEV)
        static.copy_(v)
        graph.replay()
        eager = block(v)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), seed


# ------------------------------------------------------------------ every tile, ragged rows, neighbours, large arrays
# Rows an expert has and columns in all choose the tile (32, 64 or 128 rows) and the fp32 products' form: sizes on both
# sides of each choice, and widths that are odd, even and multiples of four.
TILES = [(300, 331, 85, 8, 2), (300, 334, 86, 8, 2), (500, 70, 44, 8, 2), (1200, 640, 336, 30, 2), (1300, 642, 334, 20, 1),
         (2000, 515, 330, 3, 2), (2000, 516, 332, 3, 2), (16100, 1042, 22, 3, 1), (16100, 1043, 23, 3, 1),
         (9000, 22, 1042, 3, 2), (20, 16, 8, 512, 64), (10, 24, 12, 40, 20)]


@pytest.mark.parametrize("rows,width,hidden,experts,k", TILES)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_products_of_every_tile(rows, width, hidden, experts, k, dtype):
    test_products_and_gradients(rows, width, hidden, experts, k, dtype)


@pytest.mark.parametrize("rows,width,hidden,experts,k", [(300, 334, 86, 8, 2), (2000, 516, 332, 3, 2), (16100, 1044, 24, 3, 1),
                                                         (9000, 22, 1042, 3, 2), (2000, 515, 331, 3, 2), (16100, 1043, 24, 3, 1)])
def test_8_bits_of_every_tile(rows, width, hidden, experts, k):
    test_products_in_8_bits(rows, width, hidden, experts, k)


# A handful of slots, each output a dot product: rows of fewer than 16 bytes, of one read and of several, odd and even.
HANDFUL = [(1, 331, 203, 9, 1), (30, 70, 46, 64, 2), (3, 5, 3, 8, 2), (4, 1, 1, 3, 2), (6, 13, 200, 16, 2), (2, 1100, 520, 4, 3),
           (8, 17, 15, 1, 1), (3, 259, 131, 60, 20)]


@pytest.mark.parametrize("rows,width,hidden,experts,k", HANDFUL)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_products_of_a_handful(rows, width, hidden, experts, k, dtype):
    test_products_and_gradients(rows, width, hidden, experts, k, dtype)


@pytest.mark.parametrize("rows,width,hidden,experts,k", HANDFUL)
def test_8_bits_of_a_handful(rows, width, hidden, experts, k):
    test_products_in_8_bits(rows, width, hidden, experts, k)


@pytest.mark.parametrize("rows,width,hidden,experts,k", [(3, 70, 46, 4, 2), (3, 71, 45, 4, 2), (12, 70, 46, 4, 2), (150, 70, 46, 4, 2), (150, 71, 45, 4, 2), (700, 331, 202, 3, 2)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_ragged_rows_do_not_reach_into_the_next(rows, width, hidden, experts, k, dtype):
    """Not-a-numbers in the rows, the gradients' rows and the experts beside: what is read past a row's end counts for
    nothing, forward and backward."""
    dt = DT[dtype]
    x, index, weight, w_in, w_out, dy = problem(rows, width, hidden, experts, k, dt, rows, empty=False)
    index = index.clamp(max=experts - 2)                # nobody has the last expert; a row may have one twice
    leaf = [t.double().requires_grad_(True) for t in (x, weight)]
    y0 = O.expert_mlp(leaf[0], index, leaf[1], w_in, w_out)
    dx0, dw0 = torch.autograd.grad(y0, leaf, dy.double())
    bad = torch.arange(rows) % 3 == 1
    x[bad], dy[bad] = float("nan"), float("nan")
    w_in[-1], w_out[-1] = float("nan"), float("nan")
    dev = [t.to(DEV).requires_grad_(True) for t in (x, weight)]
    y = X().expert_mlp(dev[0], index.to(DEV), dev[1], w_in.to(DEV), w_out.to(DEV))
    dx, dw = torch.autograd.grad(y, dev, dy.to(DEV))
    ok = ~bad
    close(y[ok.to(DEV)], y0[ok], TOL[dt], "y")
    close(dx[ok.to(DEV)], dx0[ok], TOL[dt], "dx")
    close(dw[ok.to(DEV)], dw0[ok], TOL[dt], "dweight")
    assert torch.isnan(y[bad.to(DEV)]).all()


@pytest.mark.parametrize("rows,width,hidden,experts", [(3000, 40, 24, 3), (6000, 24, 8, 70), (2600, 1100, 1060, 2)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_weight_gradients_of_uneven_experts(rows, width, hidden, experts, dtype):
    """One expert with most rows, some with a few, some with none: positions dealt out in shares, whole and partial."""
    dt = DT[dtype]
    x, _, weight, w_in, w_out, dy = problem(rows, width, hidden, experts, 1, dt, rows, empty=False)
    index = torch.where(torch.rand(rows, generator=gen(1)) < 0.9, experts - 1, torch.randint(0, max(1, experts // 2), (rows,), generator=gen(2)))
    index = index.int().unsqueeze(1)
    leaf = [t.double().requires_grad_(True) for t in (w_in, w_out)]
    ref = torch.autograd.grad(O.expert_mlp(x, index, weight, leaf[0], leaf[1]), leaf, dy.double())
    dev = [t.to(DEV).requires_grad_(True) for t in (w_in, w_out)]
    runs = [torch.autograd.grad(X().expert_mlp(x.to(DEV), index.to(DEV), weight.to(DEV), *dev), dev, dy.to(DEV)) for _ in range(2)]
    for a, b, r, n in zip(*runs, ref, ("dw_in", "dw_out")):
        assert torch.equal(a, b)
        close(a, r, TOL[dt], n)


def test_products_of_very_different_sizes_by_tiles():
    """As test_products_of_very_different_sizes, where the fp32 products scale each row and column."""
    x, index, weight, w_in, w_out, dy = problem(900, 96, 64, 3, 1, torch.float32, 8, empty=False)
    x = x * torch.exp2(torch.linspace(-30, 10, 900)).unsqueeze(1)
    dy = dy * torch.exp2(torch.linspace(20, -25, 900)).unsqueeze(1)
    leaf = x.double().requires_grad_(True)
    y0 = O.expert_mlp(leaf, index, weight, w_in, w_out)
    dx0, = torch.autograd.grad(y0, leaf, dy.double())
    xd = x.to(DEV).requires_grad_(True)
    y = X().expert_mlp(xd, index.to(DEV), weight.to(DEV), w_in.to(DEV), w_out.to(DEV))
    dx, = torch.autograd.grad(y, xd, dy.to(DEV))
    for a, b in ((y, y0), (dx, dx0)):
        err = (a.detach().double().cpu() - b.detach()).abs().amax(1) / b.detach().abs().amax(1)
        assert float(err.max()) < 1e-5


def test_rows_far_apart():
    """Row strides that put the last rows past 2^32 bytes."""
    hold = torch.empty(300 * 4_000_004, device=DEV)      # 4.8 GB
    for rows, stride in ((300, 4_000_004), (40, 30_000_004)):
        x, index, weight, w_in, w_out, dy = problem(rows, 64, 40, 4, 2, torch.float32, rows)
        v = hold.as_strided((rows, 64), (stride, 1))
        v.copy_(x)
        y0 = O.expert_mlp(x, index, weight, w_in, w_out)
        close(X().expert_mlp(v, index.to(DEV), weight.to(DEV), w_in.to(DEV), w_out.to(DEV)), y0, TOL[torch.float32])
        norm, _ = X().rms_norm(v, torch.ones(64, device=DEV))
        close(norm, x.double() * (x.double().square().mean(1, keepdim=True) + 1e-6).rsqrt(), 1e-6, "norm")
        idx, w = X().route_experts(v, 3)
        assert torch.equal(idx.cpu().long(), x.topk(3, dim=1).indices)


def test_rows_of_more_than_four_gigabytes():
    """Rows that no buffer of 32-bit offsets holds, contiguous: values are read one by one through 64-bit addresses."""
    rows, width, hidden = 1_100_000, 1000, 8
    x = torch.empty(rows, width, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    index = (torch.arange(rows, device=DEV, dtype=torch.int32) * 7 % 5 - 1).unsqueeze(1)   # experts 0 to 3 and none
    weight = torch.rand(rows, 1, device=DEV) + 0.5
    g = gen(3)
    w_in = (rn(g, 4, 2 * hidden, width) / math.sqrt(width)).float()
    w_out = (rn(g, 4, width, hidden) / math.sqrt(hidden)).float()
    xd = x.requires_grad_(True)
    y = X().expert_mlp(xd, index, weight, w_in.to(DEV), w_out.to(DEV))
    dx, = torch.autograd.grad(y, xd, x.detach())
    some = torch.cat([torch.arange(0, 50), torch.arange(rows - 300, rows), torch.arange(536_000, 537_200)])
    leaf = x.detach()[some.to(DEV)].cpu().double().requires_grad_(True)
    y0 = O.expert_mlp(leaf, index[some.to(DEV)].cpu(), weight[some.to(DEV)].cpu(), w_in, w_out)
    dx0, = torch.autograd.grad(y0, leaf, leaf.detach())
    close(y.detach()[some.to(DEV)], y0, TOL[torch.float32], "y")
    close(dx[some.to(DEV)], dx0, TOL[torch.float32], "dx")


def test_more_rows_than_a_launch():
    rows = (1 << 23) + 5
    x = torch.randn(rows, 2, device=DEV)
    y, rstd = X().rms_norm(x, torch.ones(2, device=DEV))
    want = x.double() * (x.double().square().mean(1, keepdim=True) + 1e-6).rsqrt()
    assert float((y - want).abs().max()) < 1e-6
    codes, scale, _ = X().rms_norm_q8(x, torch.ones(2, device=DEV))
    assert float((codes * scale.unsqueeze(1) - want).abs().max()) < 1.5 / 127
    rows = (1 << 24) + 3
    l = torch.randn(rows, 3, device=DEV)
    index, weight = X().route_experts(l, 1)
    # the choice has the largest score to the last bits of 32, as in test_route (logits one bit apart share a score)
    s = l.double().softmax(1)
    assert float((s.max(1).values - s.gather(1, index.long())[:, 0]).max()) <= 4e-7
    assert float((weight - 1).abs().max()) < 1e-6
