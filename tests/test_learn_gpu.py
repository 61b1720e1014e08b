"""Operators of the training step on the GPU against 64 bits (oracle/learn.py).

Tolerances: an output in 32 bits is a sum of terms, off by at most k 2^-24 times the sum of their magnitudes, k the
number of roundings a term goes through: at most 40 elementwise ones and those of the sum, one for each value a thread
adds (width / 64 within a row, rows over the rows) and ten of the tree.  bfloat16 outputs are off by half a step, 2^-8 of
the value, more."""

import itertools
import math

import numpy as np
import pytest
import torch

from fsctep_amd import learn_ops as L, optim
from oracle import learn as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
EPS = 1e-5


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def close(got, want, size, k, what):
    """Within k roundings of 32 bits, and one of the output's type."""
    tol = k * U * size + (2.0 ** -8 * want.abs() if got.dtype == BF16 else 0) + 1e-37
    off = (got.double() - want).abs()
    assert got.shape == want.shape, what
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float((off / tol).max()):.3g} of its bound"


# ------------------------------------------------------------------ layer norm
def norm_call(x, w, b, silu, dy, v, vw=None, vb=None):
    x, dy = x.detach().requires_grad_(True), dy.detach().requires_grad_(True)
    ins = {"x": x} | {k: t.detach().requires_grad_(True) for k, t in (("w", w), ("b", b)) if t is not None}
    y = L.layer_norm(x, ins.get("w"), ins.get("b"), EPS, "silu" if silu else None)
    out = {"y": y}
    first = dict(zip(ins, torch.autograd.grad(y, list(ins.values()), dy, create_graph=True)))
    out |= {"d" + k: g for k, g in first.items()}
    ends = [(first["x"], v)] + [(first[k], c) for k, c in (("w", vw), ("b", vb)) if c is not None]
    ins["dy"] = dy
    second = torch.autograd.grad([e for e, _ in ends], list(ins.values()), [c for _, c in ends], allow_unused=True)
    out |= {"g" + k: torch.zeros_like(t) if g is None else g for (k, t), g in zip(ins.items(), second)}
    return {k: t.detach() for k, t in out.items()}


def norm_check(x, w, b, silu, dy, v, vw=None, vb=None):
    got = norm_call(x, w, b, silu, dy, v, vw, vb)
    want = O.norm_all(x, w, b, EPS, silu, dy, v, vw, vb)
    size = O.norm_sizes(x, w, b, EPS, silu, dy, v, vw, vb)
    rows, width = x.shape
    assert got.keys() == want.keys()
    for name, t in got.items():
        k = 50 + width / 64 + (rows if name in ("dw", "db", "gw", "gb") else 0)
        close(t, want[name], size[name], k, f"{name} of {rows} x {width}")


def norm_inputs(rows, width, dtype, wtype, seed=0):
    g = gen(1000 * rows + width + seed)
    x = torch.exp(0.5 * randn(g, rows, 1)) * (randn(g, rows, width) + randn(g, rows, 1))
    return dict(x=x.to(dtype), w=(1 + 0.3 * randn(g, width)).to(wtype), b=(0.2 * randn(g, width)).to(wtype),
                dy=randn(g, rows, width, dtype=dtype), v=randn(g, rows, width, dtype=dtype),
                vw=randn(g, width, dtype=wtype), vb=randn(g, width, dtype=wtype))


SIZES = [(1, 65), (3, 128), (33, 96), (7, 100), (130, 331), (9, 640), (3, 1600), (2, 2048), (2, 2049), (3, 4100), (1, 9001),
         (4099, 128), (1030, 67)]


@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("dtype,wtype", [(F32, F32), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("rows,width", SIZES)
def test_layer_norm(rows, width, dtype, wtype, silu):
    norm_check(silu=silu, **norm_inputs(rows, width, dtype, wtype))


@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width", [(1, 1), (5, 1), (4, 2), (7, 3), (65, 8), (9, 17), (200, 33), (3, 64)])
def test_narrow_rows(rows, width, dtype, silu):
    """At most 64 values a row, where a gradient is what is left of nearly equal numbers: values in 64 bits, rounded
    once.  What is left of them in 64 bits itself is 2^-53 of the terms' size, 2^-24 of which is far above."""
    a = norm_inputs(rows, width, dtype, dtype)
    got, want = norm_call(silu=silu, **a), O.norm_all(eps=EPS, silu=silu, **a)
    size = O.norm_sizes(eps=EPS, silu=silu, **a)
    for name, t in got.items():
        k = rows + 50 if name in ("dw", "db", "gw", "gb") else 50 if name == "y" else 2 ** -10
        tol = k * U * size[name] + (2.0 ** -8 if dtype == BF16 else U * 4) * want[name].abs() + 1e-37
        assert ((t.double() - want[name]).abs() <= tol).all(), name


@pytest.mark.parametrize("rows,width", [(1, 4097), (3, 4100), (5, 5001), (40, 6144), (2, 8191), (600, 8192), (3, 8193), (2, 12001)])
@pytest.mark.parametrize("dtype,silu", [(F32, False), (F32, True), (BF16, True)])
def test_wide_rows(rows, width, dtype, silu):
    norm_check(silu=silu, **norm_inputs(rows, width, dtype, F32))


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("silu", [False, True])
def test_layer_norm_without_weight_or_bias(weight, bias, silu):
    a = norm_inputs(37, 200, F32, F32)
    if not weight:
        a["w"] = a["vw"] = None
    if not bias:
        a["b"] = a["vb"] = None
    norm_check(silu=silu, **a)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layer_norm_strides(dtype):
    """Rows of a wider array, rows from an odd address, one row many times, and transposed rows."""
    g = gen(3)
    for width in (128, 131, 1600):
        a = norm_inputs(21, width, dtype, dtype)
        wide = randn(g, 21, width + 13, dtype=dtype)
        odd = randn(g, 21 * width + 1, dtype=dtype)[1:].view(21, width)
        turned = randn(g, width, 21, dtype=dtype).t()
        same = randn(g, 1, width, dtype=dtype).expand(21, width)
        for x, dy, v in ((wide[:, 5:5 + width], odd, same), (odd, same, wide[:, 1:1 + width]), (same, turned, odd),
                         (turned, wide[:, :width], turned)):
            norm_check(silu=True, **(a | dict(x=x, dy=dy, v=v)))


def test_rows_far_from_zero():
    """A mean of 1,000 deviations: the deviations keep their accuracy (their own rounding in the input aside)."""
    a = norm_inputs(40, 640, F32, F32)
    a["x"] = a["x"] + 1000.0
    norm_check(silu=False, **a)
    norm_check(silu=True, **a)


def test_rows_of_one_value_and_of_zeros():
    for width in (16, 640):
        a = norm_inputs(6, width, F32, F32)
        a["x"] = a["x"].clone()
        a["x"][0] = 0.0
        a["x"][1] = 7.25
        norm_check(silu=True, **a)


@pytest.mark.parametrize("width", [48, 640, 2500])
def test_rows_with_nan_and_infinities_stay_apart(width):
    a = norm_inputs(9, width, F32, F32)
    clean = norm_call(silu=True, **(a | dict(vw=None, vb=None)))
    x = a["x"].clone()
    x[2, 3], x[5, 0], x[7, width - 1] = math.nan, math.inf, -math.inf
    got = norm_call(silu=True, **(a | dict(x=x, vw=None, vb=None)))
    bad = [2, 5, 7]
    rest = [i for i in range(9) if i not in bad]
    for name in ("y", "dx", "gx", "gdy"):
        assert got[name][bad].isnan().all(), name
        assert torch.equal(got[name][rest], clean[name][rest]), name
    for name in ("dw", "gw", "gb"):
        assert got[name].isnan().all(), name


def test_silu_at_large_arguments():
    """Rows whose normalised values reach the sigmoid's ends: no NaN where 0 times infinity lies near."""
    a = norm_inputs(5, 300, F32, F32)
    a["w"] = a["w"] * 3000
    got, want = norm_call(silu=True, **a), O.norm_all(eps=EPS, silu=True, **a)
    for name in got:
        assert torch.isfinite(got[name]).all(), name
    close(got["y"], want["y"], O.norm_sizes(eps=EPS, silu=True, **a)["y"], 100, "y")


@pytest.mark.parametrize("rows,width", [(40, 20), (33, 128), (9, 331), (300, 640), (7, 1600), (3, 3000)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_both_gradients_of_a_force_loss(rows, width, dtype):
    """A loss of the rows' output and of their gradient: what reaches x by the two ways is the sum of the two, and either way
    alone is there without the other; weight and bias that need no gradient change nothing."""
    a = norm_inputs(rows, width, dtype, dtype)
    g = gen(rows)
    ey = randn(g, rows, width, dtype=dtype)

    def grads(ends, needs):
        x, dy = a["x"].detach().requires_grad_(True), a["dy"].detach().requires_grad_(True)
        w, b = (a[k].detach().requires_grad_(needs) for k in ("w", "b"))
        y = L.layer_norm(x, w, b, EPS, "silu")
        dx, = torch.autograd.grad(y, x, dy, create_graph=True)
        pick = {"dx": (dx, a["v"]), "y": (y, ey)}
        outs = [pick[e] for e in ends]
        ins = [x, w, b] if needs else [x]
        return torch.autograd.grad([o for o, _ in outs], ins, [c for _, c in outs])

    one, two, both = grads(["dx"], True), grads(["y"], True), grads(["dx", "y"], True)
    size = O.norm_sizes(a["x"], a["w"], a["b"], EPS, True, a["dy"], a["v"])
    other = O.norm_sizes(a["x"], a["w"], a["b"], EPS, True, ey, a["v"])
    for k, (p, q, s) in enumerate(zip(one, two, both)):
        # each part and their sum are rounded to the type, x's sum once: half a step of each of the three
        step = 2.0 ** -8 if dtype == BF16 else U
        terms = (p.double().abs() + q.double().abs() + s.double().abs()) * step
        name = ("gx", "gw", "gb")[k], ("dx", "dw", "db")[k]
        assert ((p.double() + q.double() - s.double()).abs() <= terms + 4 * U * (size[name[0]] + other[name[1]])).all(), name
    for ends in (["dx"], ["y"], ["dx", "y"]):
        assert torch.equal(grads(ends, False)[0], grads(ends, True)[0])


def test_any_part_of_both_gradients():
    """Every choice of the ends of a force loss and of the leaves asked for, against 64 bits; a weight or bias that needs no
    gradient, or is not there."""
    a = norm_inputs(37, 150, F32, F32)
    g = gen(5)
    ey, ew = randn(g, 37, 150), randn(g, 150)

    def grads(norm, t, ends, first, ask, frozen):
        leaf = {k: v.detach().requires_grad_(k not in frozen) for k, v in t.items() if k in ("x", "w", "b", "dy") and "no " + k not in frozen}
        y = norm(leaf["x"], leaf.get("w"), leaf.get("b"))
        d = dict(zip(first, torch.autograd.grad(y, [leaf[k] for k in first], leaf["dy"], create_graph=True)))
        out = {"y": (y, t["ey"])} | {"d" + k: (d[k], t["c" + k]) for k in first}
        pairs = [out[e] for e in ends if e in out]
        return torch.autograd.grad([p for p, _ in pairs], [leaf[k] for k in ask], [c for _, c in pairs], allow_unused=True)

    t = {"x": a["x"], "w": a["w"], "b": a["b"], "dy": a["dy"], "ey": ey, "cx": a["v"], "cw": ew, "cb": a["vb"]}
    wide = {k: v.double() for k, v in t.items()}
    mine = lambda x, w, b: L.layer_norm(x, w, b, EPS, "silu")  # noqa: E731
    plain = lambda x, w, b: O.layer_norm(x, w, b, EPS, True)  # noqa: E731
    for frozen in ((), ("w",), ("b",), ("no w",), ("no b",), ("no w", "no b"), ("x",)):
        have = [k for k in ("x", "w", "b") if k not in frozen and "no " + k not in frozen]
        for first in ([k for k in have if k == "x"], have, have[-1:]):
            for ends in (["y"], ["d" + k for k in first], ["y"] + ["d" + k for k in first]):
                for ask in (have, have[:1], have[-1:], have + ["dy"]):
                    if not first:
                        continue
                    got, want = grads(mine, t, ends, first, ask, frozen), grads(plain, wide, ends, first, ask, frozen)
                    for k, p, q in zip(ask, got, want):
                        what = (frozen, first, ends, ask, k)
                        p = torch.zeros_like(t[k]) if p is None else p
                        q = torch.zeros_like(wide[k]) if q is None else q
                        # terms of order 1, 10 at most after the weights: sums of 150 and 37 of them
                        assert float((p.double() - q).abs().max()) <= 400 * U * 10 * max(1.0, float(q.abs().max())), what


def test_gradients_of_weight_and_bias_alone():
    """Rows that need no gradient."""
    a = norm_inputs(50, 200, F32, F32)
    w, b, dy = (a[k].detach().requires_grad_(True) for k in ("w", "b", "dy"))
    y = L.layer_norm(a["x"], w, b, EPS, "silu")
    dw, db = torch.autograd.grad(y, (w, b), dy, create_graph=True)
    got = torch.autograd.grad((dw, db, y), (w, b, dy), (a["vw"], a["vb"], a["v"]), allow_unused=True)
    w6, b6, dy6 = (a[k].detach().double().requires_grad_(True) for k in ("w", "b", "dy"))
    y6 = O.layer_norm(a["x"].double(), w6, b6, EPS, True)
    dw6, db6 = torch.autograd.grad(y6, (w6, b6), dy6, create_graph=True)
    want = torch.autograd.grad((dw6, db6, y6), (w6, b6, dy6), (a["vw"].double(), a["vb"].double(), a["v"].double()))
    for p, q in zip(got, want):
        assert float((p.double() - q).abs().max()) <= 200 * U * max(1.0, float(q.abs().max()))


def test_no_rows():
    x, w, b = torch.zeros(0, 70, device=DEV), torch.ones(70, device=DEV), torch.zeros(70, device=DEV)
    got = norm_call(x, w, b, True, x, x, w, b)
    assert got["y"].shape == (0, 70) and all(float(got[k].abs().sum()) == 0 for k in ("dw", "db", "gw", "gb"))


def test_forward_without_gradients_keeps_nothing():
    x = torch.randn(5, 70, device=DEV)
    y, mean, rstd = torch.ops.fsctep.layer_norm(x, None, None, EPS, 0, False)
    assert mean.numel() == rstd.numel() == 0
    with torch.no_grad():
        assert torch.equal(L.layer_norm(x), y)


def test_layer_norm_repeats_to_the_bit():
    a = norm_inputs(5000, 331, F32, F32)
    one, two = norm_call(silu=True, **a), norm_call(silu=True, **a)
    assert all(torch.equal(one[k], two[k]) for k in one)


def test_layer_norm_gradient_against_differences():
    """A central difference of step h along a unit direction is off by h^2 / 6 third derivatives (a few units of the row
    sum here) and by the values' own roundings over h: 2^-24 |y| sum / h."""
    for silu in (False, True):
        a = norm_inputs(4, 96, F32, F32)
        g = gen(9)
        d, h = randn(g, 4, 96), 2.0 ** -6
        d = d / d.norm()
        x = a["x"].clone().requires_grad_(True)
        call = lambda t: (L.layer_norm(t, a["w"], a["b"], EPS, "silu" if silu else None).double() * a["dy"].double()).sum()  # noqa: E731
        dx, = torch.autograd.grad(call(x), x)
        with torch.no_grad():
            diff = (call(x + h * d) - call(x - h * d)) / (2 * h)
            size = (L.layer_norm(x, a["w"], a["b"]).abs() * a["dy"].abs()).double().sum()
        assert abs(float((dx.double() * d).sum() - diff)) <= 20 * h * h + 8 * U * float(size) / h


def test_second_gradient_against_differences():
    """The gradient of (dx . v) along a direction against differences of dx, the same bound."""
    a = norm_inputs(4, 96, F32, F32)
    g = gen(10)
    d, h = randn(g, 4, 96), 2.0 ** -6
    d = d / d.norm()

    def dx_of(t, create):
        t = t.detach().requires_grad_(True)
        y = L.layer_norm(t, a["w"], a["b"], EPS, "silu")
        return t, torch.autograd.grad(y, t, a["dy"], create_graph=create)[0]

    x, dx = dx_of(a["x"], True)
    gx, = torch.autograd.grad(dx, x, a["v"])
    diff = ((dx_of(x + h * d, False)[1] - dx_of(x - h * d, False)[1]).double() * a["v"].double()).sum() / (2 * h)
    size = float((dx.double().abs() * a["v"].double().abs()).sum())
    assert abs(float((gx.double() * d).sum() - diff)) <= 40 * h * h + 40 * U * size / h


# ------------------------------------------------------------------ lookup
def tokens(g, rows, table, index_type, kind):
    if kind == "one":
        at = torch.full((rows,), table // 2, device=DEV)
    elif kind == "tail":
        at = (torch.exp(torch.rand(rows, generator=g, device=DEV) * math.log(table + 1.0)) - 1).long().clamp(max=table - 1)
    elif kind == "sorted":
        at = torch.sort(torch.randint(0, table, (rows,), generator=g, device=DEV))[0]
    else:
        at = torch.randint(0, table, (rows,), generator=g, device=DEV)
    if kind == "outside" and rows > 3:
        at[::3] = -1
        at[1] = table
        at[2] = 2 ** 40 if index_type == torch.int64 else 2 ** 31 - 1
        at[rows - 1] = -2 ** 31
    return at.to(index_type)


LOOKUPS = [(0, 5, 7), (1, 1, 1), (1, 16, 100), (32, 16, 100), (64, 3, 2), (65, 4, 300), (257, 64, 1), (300, 331, 40),
           (1000, 130, 257), (4097, 192, 9), (5000, 40, 70000), (20000, 7, 12), (70001, 20, 300), (9000, 1025, 3),
           (130, 12288, 5), (40000, 2, 5000)]


def lookup_check(table, index, scale, dy):
    t = table.detach().requires_grad_(True)
    y = L.embedding(t, index, scale)
    want = O.embedding(table.double(), index, scale)
    close(y, want, want.abs(), 2, "rows")         # the scale's rounding and the product's
    dt, = torch.autograd.grad(y, t, dy)
    flat, d2 = index.reshape(-1), dy.reshape(-1, dy.shape[-1])
    want = O.embedding_grad(d2, flat, table.shape[0], scale)
    size = O.embedding_grad(d2.abs(), flat, table.shape[0], abs(scale))
    close(dt, want, size, 4 + math.sqrt(flat.numel()) + min(flat.numel(), 600), "dtable")
    return y, dt


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind,index_type", [("free", torch.int64), ("one", torch.int32), ("tail", torch.int64),
                                             ("sorted", torch.int32), ("outside", torch.int64), ("outside", torch.int32)])
@pytest.mark.parametrize("rows,width,table", LOOKUPS)
def test_embedding(rows, width, table, kind, index_type, dtype):
    g = gen(rows + width + table)
    lookup_check(randn(g, table, width, dtype=dtype), tokens(g, rows, table, index_type, kind), 1.7,
                 randn(g, rows, width, dtype=dtype))


@pytest.mark.parametrize("table", [1, 23, 24, 25, 100, 255, 256, 257, 520, 65535, 65536, 65537])
@pytest.mark.parametrize("rows", [255, 256, 257, 1023, 1024, 1025, 2049, 33000])
def test_embedding_at_the_rules_borders(rows, table):
    """Where another kernel takes over: by tokens, table rows, digits of the sort, shares."""
    g = gen(rows * table)
    for dtype, width in ((F32, 36), (BF16, 75)):
        lookup_check(randn(g, table, width, dtype=dtype), tokens(g, rows, table, torch.int32, "tail"), 1.0,
                     randn(g, rows, width, dtype=dtype))


@pytest.mark.parametrize("kind", ["tail", "one", "outside"])
@pytest.mark.parametrize("rows,table", [(512, 9), (513, 9), (512, 24), (513, 24), (2048, 25), (2049, 25), (511, 2048), (65, 2049), (2048, 4096),
                                        (2048, 4097), (1024, 8193), (256, 32768), (256, 32769), (1, 70000), (7, 66000)])
def test_embedding_of_few_tokens(rows, table, kind):
    """Where one launch takes over from the sort, by tokens and by table rows, and where a block has fewer waves."""
    g = gen(rows + table)
    for dtype, width in ((F32, 36), (BF16, 75), (F32, 3)):
        lookup_check(randn(g, table, width, dtype=dtype), tokens(g, rows, table, torch.int64, kind), 0.5,
                     randn(g, rows, width, dtype=dtype))


def test_embedding_of_any_shape_and_scale():
    g = gen(1)
    t = randn(g, 20, 24)
    for shape in ((), (3,), (4, 5), (2, 3, 4)):
        index = torch.randint(0, 20, shape, generator=g, device=DEV)
        for scale in (1.0, 0.0, -2.5):
            y, _ = lookup_check(t, index, scale, randn(g, *shape, 24))
            assert y.shape == (*shape, 24)


def test_embedding_strides():
    g = gen(2)
    for dtype in (F32, BF16):
        for width in (24, 33):
            wide, index = randn(g, 30, width + 9, dtype=dtype), torch.randint(0, 30, (500,), generator=g, device=DEV)
            dys = (randn(g, 500, width + 3, dtype=dtype)[:, 2:2 + width], randn(g, 1, width, dtype=dtype).expand(500, width),
                   randn(g, width, 500, dtype=dtype).t(), randn(g, 500 * width + 1, dtype=dtype)[1:].view(500, width))
            for dy in dys:
                lookup_check(wide[:, 3:3 + width], index, 1.0, dy)
            lookup_check(wide[:, 3:3 + width], torch.randint(0, 30, (1000,), generator=g, device=DEV)[::2], 1.0, dys[0])
            lookup_check(randn(g, width, 30, dtype=dtype).t(), index, 1.0, dys[0])


def test_no_table():
    t = torch.zeros(0, 6, device=DEV).requires_grad_(True)
    y = L.embedding(t, torch.zeros(4, dtype=torch.long, device=DEV))
    assert float(y.abs().sum()) == 0 and torch.autograd.grad(y.sum(), t)[0].shape == (0, 6)


def test_embedding_outside_rows_ignore_what_stands_there():
    """Tokens outside the table give zeros even from a table of NaN, and rows of dy that they name do not count."""
    t = torch.full((4, 40), math.nan, device=DEV).requires_grad_(True)
    index = torch.tensor([-1, 4, 2, -1], device=DEV)
    y = L.embedding(t, index)
    assert (y[[0, 1, 3]] == 0).all() and y[2].isnan().all()
    dy = torch.ones(4, 40, device=DEV)
    dy[[0, 1, 3]] = math.nan
    dt, = torch.autograd.grad(y, t, dy)
    assert (dt[2] == 1).all() and (dt[[0, 1, 3]] == 0).all()


def test_embedding_repeats_to_the_bit():
    g = gen(4)
    for rows, table in ((50000, 9), (50000, 40000), (700, 20)):
        t, index = randn(g, table, 100).requires_grad_(True), torch.randint(0, table, (rows,), generator=g, device=DEV)
        dy = randn(g, rows, 100)
        one, two = (torch.autograd.grad(L.embedding(t, index), t, dy)[0] for _ in range(2))
        assert torch.equal(one, two)


def test_embedding_differentiates_to_any_order():
    g = gen(5)
    t, index = randn(g, 11, 20).requires_grad_(True), torch.randint(-1, 11, (400,), generator=g, device=DEV)
    dy, c = randn(g, 400, 20).requires_grad_(True), randn(g, 11, 20)
    y = L.embedding(t, index, 3.0)
    dt, = torch.autograd.grad(y ** 3, t, dy, create_graph=True)
    gt, gdy = torch.autograd.grad(dt, (t, dy), c, create_graph=True)
    third, = torch.autograd.grad(gt.sum(), t)
    with torch.enable_grad():
        t6, dy6 = t.detach().double().requires_grad_(True), dy.detach().double().requires_grad_(True)
        dt6, = torch.autograd.grad(O.embedding(t6, index, 3.0) ** 3, t6, dy6, create_graph=True)
        gt6, gdy6 = torch.autograd.grad(dt6, (t6, dy6), c.double(), create_graph=True)
        third6, = torch.autograd.grad(gt6.sum(), t6)
    for a, b in ((dt, dt6), (gt, gt6), (gdy, gdy6), (third, third6)):
        assert float((a.double() - b).abs().max()) <= 400 * U * float(b.abs().max())


def test_lookup_past_32_bits():
    """Offsets past 2^32 bytes and 2^31 values in the rows, and past 2^31 values in the table."""
    rows, width = 1_100_000, 2048
    index = torch.arange(rows, device=DEV) % 7
    t = randn(gen(6), 7, width, dtype=BF16).requires_grad_(True)
    y = L.embedding(t, index)
    for i in (0, 5, rows - 1):
        assert torch.equal(y[i], t[i % 7])
    dy = torch.zeros(rows, width, dtype=BF16, device=DEV)
    dy[rows - 1], dy[rows - 9] = 1.0, 2.0
    dt, = torch.autograd.grad(y, t, dy)
    want = torch.zeros(7, device=DEV)
    want[(rows - 1) % 7] += 1
    want[(rows - 9) % 7] += 2
    assert torch.equal(dt.float(), want.unsqueeze(1).expand(7, width))
    del y, dy, dt
    big = torch.zeros(rows, width, dtype=BF16, device=DEV).requires_grad_(True)
    with torch.no_grad():
        big[rows - 2] = 3.0
    index = torch.tensor([rows - 2, 0, rows - 2], device=DEV)
    y = L.embedding(big, index)
    assert (y[0] == 3).all() and (y[1] == 0).all()
    dt, = torch.autograd.grad(y, big, torch.ones_like(y))
    assert (dt[rows - 2] == 2).all() and (dt[0] == 1).all() and float(dt.float().abs().sum()) == 3 * width


# ------------------------------------------------------------------ AdamW
def model(sizes, dtype, seed, bits=32):
    g = gen(seed)
    p = [randn(g, n) for n in sizes]
    s = dict(params=[t.to(dtype) for t in p], grads=[randn(g, n, dtype=dtype) * 10.0 ** -(i % 5) for i, n in enumerate(sizes)])
    m, r = [0.3 * t.float() for t in s["grads"]], [t.float().abs() + 1e-4 for t in s["grads"]]
    if bits == 32:
        s |= dict(exp_avgs=m, exp_avg_sqs=[t * t for t in r])
    else:
        for name, values, root in (("exp_avg", m, False), ("root", r, True)):
            coded = [O.encode(t.cpu().numpy(), 3, root) for t in values]
            s[name + "s"] = [torch.from_numpy(c).to(DEV) for c, _ in coded]
            s[name + "_scales"] = [torch.from_numpy(c).to(DEV) for _, c in coded]
    s["steps"] = [torch.full((), float(5 + i), device=DEV) for i in range(len(sizes))]
    if dtype == BF16:
        s["masters"] = p
    return s


SETS = [[1], [3, 255, 256, 257, 2048, 5000, 0, 7], [100] * 131, [70001, 2]]
RULE = dict(lr=3e-3, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.1)


def copies(s):
    return {k: [t.clone() for t in v] for k, v in s.items()}


@pytest.mark.parametrize("max_norm", [None, 0.5, 1e6])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("sizes", SETS)
def test_adamw(sizes, dtype, max_norm):
    """m and v in 3 and 4 roundings, p in 8 of terms of at most |p| and the step's size, and half a step of bfloat16."""
    s = model(sizes, dtype, 1)
    old = copies(s)
    norm = optim.adamw_step(**s, max_norm=max_norm, **RULE)
    want_norm = math.sqrt(sum(float(g.double().square().sum()) for g in old["grads"]))
    clip = 1.0
    if max_norm:
        assert abs(float(norm) - want_norm) <= 2 * U * want_norm
        clip = min(1.0, max_norm / (want_norm + 1e-6))
    else:
        assert norm is None
    for i in range(len(sizes)):
        p0 = (old["masters"] if dtype == BF16 else old["params"])[i].double().cpu().numpy()
        args = [old[k][i].double().cpu().numpy() for k in ("grads", "exp_avgs", "exp_avg_sqs")]
        p, m, v = O.adamw(p0, *args, 5 + i, clip=clip, **RULE)
        size = np.abs(args[1]) + np.abs(args[0])
        assert (np.abs(s["exp_avgs"][i].double().cpu().numpy() - m) <= 6 * U * size).all()
        assert (np.abs(s["exp_avg_sqs"][i].double().cpu().numpy() - v) <= 8 * U * v + 1e-44).all()
        got = (s["masters"] if dtype == BF16 else s["params"])[i].double().cpu().numpy()
        assert (np.abs(got - p) <= 4 * U * np.abs(p0) + 16 * U * (np.abs(p - p0) + 20 * RULE["lr"])).all()
        if dtype == BF16:
            assert torch.equal(s["params"][i], s["masters"][i].to(BF16))
        assert float(s["steps"][i]) == 6 + i
        assert torch.equal(s["grads"][i], old["grads"][i])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("sizes", SETS)
def test_adamw_in_8_bits(sizes, dtype):
    """Codes and scales to the bit: every operation rounds by itself, as numpy's in float32."""
    s = model(sizes, dtype, 2, bits=8)
    old = copies(s)
    optim.adamw_step_q8(**s, **RULE)
    f = np.float32
    b1, b2 = RULE["betas"]
    for i in range(len(sizes)):
        g = old["grads"][i].float().cpu().numpy()
        m = O.decode(old["exp_avgs"][i].cpu().numpy(), old["exp_avg_scales"][i].cpu().numpy(), False)
        r = O.decode(old["roots"][i].cpu().numpy(), old["root_scales"][i].cpu().numpy(), True)
        m2 = f(b1) * m + f(1 - b1) * g
        r2 = np.sqrt(f(b2) * (r * r) + f(1 - b2) * g * g)
        for name, value, root in (("exp_avg", m2, False), ("root", r2, True)):
            code, scale = O.encode(value, 6 + i, root)
            assert np.array_equal(s[name + "_scales"][i].cpu().numpy(), scale), (name, i)
            assert np.array_equal(s[name + "s"][i].cpu().numpy(), code), (name, i)
            values = (optim.root_values if root else optim.moment_values)(s[name + "s"][i], s[name + "_scales"][i])
            assert np.array_equal(values.cpu().numpy(), O.decode(code, scale, root))
        p0 = (old["masters"] if dtype == BF16 else old["params"])[i].double().cpu().numpy()
        p, _, _ = O.adamw(p0, g.astype(np.float64), m.astype(np.float64), r.astype(np.float64) ** 2, 5 + i, **RULE)
        got = (s["masters"] if dtype == BF16 else s["params"])[i].double().cpu().numpy()
        assert (np.abs(got - p) <= 4 * U * np.abs(p0) + 16 * U * (np.abs(p - p0) + 20 * RULE["lr"])).all()


def test_8_bit_states_of_zeros_and_tiny_values():
    n = 1024
    p, g = torch.ones(n, device=DEV), torch.zeros(n, device=DEV)
    g[256:512] = 1e-33
    g[512] = 1.0
    g[768:] = torch.logspace(-30, 2, 256, device=DEV)
    codes = lambda: [torch.zeros(n, dtype=torch.uint8, device=DEV)]  # noqa: E731
    scales = lambda: [torch.zeros(n // 256, device=DEV)]  # noqa: E731
    m, ms, r, rs, t = codes(), scales(), codes(), scales(), [torch.zeros((), device=DEV)]
    for _ in range(3):
        optim.adamw_step_q8([p], [g], m, ms, r, rs, t, lr=0.1, weight_decay=0.0)
    mv, rv = optim.moment_values(m[0], ms[0]), optim.root_values(r[0], rs[0])
    assert torch.isfinite(p).all() and (p[:256] == 1).all() and (mv[:512] == 0).all() and (rv[:512] == 0).all()
    # sqrt(v) of a value above zero stays above zero, so that no step grows without bound
    assert (rv[768:][g[768:] > 1e-18] > 0).all()
    assert float((p - 1).abs().max()) <= 3 * 0.1 * 1.7


def test_8_bit_states_follow_the_32_bit_ones():
    """Gradients of a fixed spread over 400 steps: sqrt(v) of the codes stays near that of 32 bits.  A rounding to a grid of
    share s = 1 / 16 moves v by a random s sqrt(f (1 - f)) of twice the root, f the place between neighbours; with
    steps of 0.05 of v (beta2 = 0.95) its stationary scatter is at most 2 s / 2 / sqrt(2 * 0.05) = 0.2 of v, 0.1 of the root,
    and the mean over 65,536 values is 0.1 / 256: ten times that, and the mean bias of a root's curvature, 0.1^2 / 2."""
    n = 65536
    g = gen(7)
    a = [torch.zeros(n, device=DEV) for _ in range(3)]
    p8, m8, r8 = torch.zeros(n, device=DEV), torch.zeros(n, dtype=torch.uint8, device=DEV), torch.zeros(n, dtype=torch.uint8, device=DEV)
    ms, rs = torch.zeros(n // 256, device=DEV), torch.zeros(n // 256, device=DEV)
    t32, t8 = torch.zeros((), device=DEV), torch.zeros((), device=DEV)
    spread = torch.exp(randn(g, n))
    for _ in range(400):
        grad = spread * randn(g, n)
        optim.adamw_step([a[0]], [grad], [a[1]], [a[2]], [t32], betas=(0.9, 0.95))
        optim.adamw_step_q8([p8], [grad], [m8], [ms], [r8], [rs], [t8], betas=(0.9, 0.95))
    ratio = optim.root_values(r8, rs).double() / a[2].double().sqrt()
    assert abs(float(ratio.mean()) - 1) <= 10 * 0.1 / 256 + 0.1 ** 2 / 2
    assert float(ratio.std()) <= 0.2


def test_adamw_unaligned_tensors_and_gradients_of_any_stride():
    g = gen(8)
    for bits in (32, 8):
        buf = {k: randn(g, 4000) for k in "pgmv"}
        for off in (1, 2, 3):
            n = 1501
            view = {k: b[off:off + n].clone().abs() for k, b in buf.items()}
            odd = {k: torch.cat([b.new_zeros(off), b])[off:] for k, b in view.items()}
            if bits == 32:
                call = lambda d: optim.adamw_step([d["p"]], [d["g"]], [d["m"]], [d["v"]], [torch.zeros((), device=DEV)])  # noqa: E731
            else:
                codes = [torch.zeros(n + off, dtype=torch.uint8, device=DEV)[off:] for _ in range(4)]
                it = iter(codes)
                call = lambda d: optim.adamw_step_q8([d["p"]], [d["g"]], [next(it)], [torch.zeros(6, device=DEV)], [next(it)],  # noqa: E731
                                                     [torch.zeros(6, device=DEV)], [torch.zeros((), device=DEV)])
            call(view)
            call(odd)
            assert all(torch.equal(view[k], odd[k]) for k in view)
    p, grad = randn(g, 40, 30), randn(g, 30, 40)
    a, b = p.clone(), p.clone()
    z = lambda: [torch.zeros(40, 30, device=DEV)]  # noqa: E731
    optim.adamw_step([a], [grad.t()], z(), z(), [torch.zeros((), device=DEV)])
    optim.adamw_step([b], [grad.t().contiguous()], z(), z(), [torch.zeros((), device=DEV)])
    assert torch.equal(a, b)


def test_the_same_tensor_twice_is_refused():
    s = model([50, 60], F32, 3)
    for name in ("params", "exp_avgs", "steps"):
        bad = copies(s)
        other = "params" if name == "params" else name
        bad[name][1] = bad[other][0] if name == "steps" else bad[other][0]
        if name != "steps":
            for k in ("params", "grads", "exp_avgs", "exp_avg_sqs"):
                if k != name:
                    bad[k][1] = bad[k][0].clone()
        with pytest.raises(RuntimeError, match="twice"):
            optim.adamw_step(**bad)


@pytest.mark.parametrize("first,second", [("params", "params"), ("params", "grads"), ("exp_avgs", "exp_avg_sqs"), ("params", "exp_avgs"),
                                          ("steps", "params")])
def test_overlapping_tensors_are_refused(first, second):
    """Two views of one array that share a value; the same views one value further apart are taken."""
    def step(apart):
        flat = torch.zeros(1000, device="cuda")
        a = {k: [torch.zeros(100, device="cuda") for _ in range(2)] for k in ("params", "grads", "exp_avgs", "exp_avg_sqs")}
        a["steps"] = [torch.zeros((), device="cuda") for _ in range(2)]
        n = a[first][0].numel()
        a[first][0] = flat[:n].view(a[first][0].shape)
        a[second][1] = flat[n - 1 + apart:n - 1 + apart + a[second][1].numel()].view(a[second][1].shape)
        optim.adamw_step(*(a[k] for k in ("params", "grads", "exp_avgs", "exp_avg_sqs", "steps")))

    step(1)
    with pytest.raises(RuntimeError, match="overlap"):
        step(0)


def test_parameters_may_share_a_gradient():
    p = [torch.full((300,), 2.0, device="cuda") for _ in range(2)]
    g = torch.linspace(-1.0, 1.0, 300, device="cuda")
    z = lambda: [torch.zeros(300, device="cuda") for _ in range(2)]
    optim.adamw_step(p, [g, g], z(), z(), [torch.zeros((), device="cuda") for _ in range(2)])
    assert torch.equal(p[0], p[1]) and not torch.equal(p[0], torch.full_like(p[0], 2.0))


def test_nan_gradients_pass_into_the_parameters():
    for max_norm in (None, 1.0):
        s = model([600, 700], F32, 4)
        s["grads"][0][3] = math.nan
        optim.adamw_step(**s, max_norm=max_norm)
        assert s["params"][0][3].isnan() and bool(s["params"][1].isnan().all()) == (max_norm is not None)


def test_optimiser_follows_torch():
    """Ten steps beside torch.optim.AdamW in 64 bits, two groups, clipped; a parameter without a gradient stays."""
    g = gen(11)
    shapes = [(33, 17), (17,), (5, 5, 5), (1,), (9,)]
    mine = [torch.nn.Parameter(randn(g, *s)) for s in shapes]
    theirs = [torch.nn.Parameter(p.detach().double()) for p in mine]
    groups = lambda ps: [dict(params=ps[:2], weight_decay=0.2), dict(params=ps[2:], lr=5e-3)]  # noqa: E731
    a = optim.AdamW(groups(mine), lr=1e-2, max_norm=2.0)
    b = torch.optim.AdamW(groups(theirs), lr=1e-2)
    for step in range(10):
        for p, q in zip(mine[:4], theirs[:4]):
            p.grad = randn(g, *p.shape)
            q.grad = p.grad.double()
        norm = torch.nn.utils.clip_grad_norm_(theirs, 2.0)
        a.step()
        b.step()
        assert abs(float(a.grad_norm) - float(norm)) <= 2 * U * float(norm)
    for p, q in zip(mine, theirs):
        # ten steps of at most 16 roundings of the parameter's and the step's size
        assert float((p.double() - q).abs().max()) <= 160 * U * (float(q.abs().max()) + 1e-2)
    assert mine[4] not in a.state
    # its state goes into torch's optimiser and back
    c = torch.optim.AdamW(groups(mine), lr=1e-2)
    c.load_state_dict(a.state_dict())
    d = optim.AdamW(groups(mine), lr=1e-2, max_norm=2.0)
    d.load_state_dict(c.state_dict())
    for p in mine[:4]:
        for k in ("step", "exp_avg", "exp_avg_sq"):
            assert torch.equal(d.state[p][k], a.state[p][k]) and d.state[p][k].device == p.device, k


@pytest.mark.parametrize("bits", [32, 8])
def test_optimiser_state_is_saved_and_loaded(bits):
    g = gen(12)
    ps = [torch.nn.Parameter(randn(g, 300).to(BF16)), torch.nn.Parameter(randn(g, 77))]
    opt = optim.AdamW(ps, lr=1e-2, state_bits=bits)
    grads = [randn(g, *p.shape, dtype=p.dtype) for p in ps]
    for p, t in zip(ps, grads):
        p.grad = t
    opt.step()
    copy = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for p, t in zip(copy, grads):
        p.grad = t
    other = optim.AdamW(copy, lr=1e-2, state_bits=bits)
    other.load_state_dict(opt.state_dict())
    for p, q in zip(ps, copy):
        assert opt.state[p].keys() == other.state[q].keys()
        for k, t in opt.state[p].items():
            assert other.state[q][k].dtype == t.dtype and torch.equal(other.state[q][k], t) and \
                other.state[q][k].data_ptr() != t.data_ptr()
    opt.step()
    other.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, copy))
    with pytest.raises(ValueError, match="bits"):
        optim.AdamW(copy, state_bits=40 - bits).load_state_dict(opt.state_dict())


def test_autograd_sees_the_step():
    """A parameter that a graph still needs may not change under it."""
    p = torch.nn.Parameter(torch.randn(50, device=DEV))
    y = (p * p).sum()
    p.grad = torch.ones_like(p)
    optim.AdamW([p]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_first_step_is_not_captured():
    """A replay would make the states anew each time."""
    p = torch.nn.Parameter(torch.randn(50, device=DEV))
    p.grad = torch.ones_like(p)
    opt = optim.AdamW([p])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="take a step before"):
        with torch.cuda.graph(graph):
            torch.zeros(1, device=DEV)
            opt.step()
    opt.step()
    assert float(opt.state[p]["step"]) == 1


def test_tensors_past_32_bits():
    """More than 2^31 values in one tensor of a step, and in the rows of a norm."""
    n = 2 ** 31 + 300
    p, g, m, v = (torch.full((n,), c, device=DEV) for c in (1.0, 0.5, 0.0, 0.0))
    step = torch.zeros((), device=DEV)
    norm = optim.adamw_step([p], [g], [m], [v], [step], lr=0.25, weight_decay=0.0, max_norm=1e9)
    assert abs(float(norm) - 0.5 * math.sqrt(n)) <= 2 * U * 0.5 * math.sqrt(n)
    # the first step's size is lr g / (|g| + eps)
    for t, c in ((p, 0.75), (m, 0.05), (v, 0.25e-3)):
        lo, hi = t.aminmax()
        assert abs(float(lo) - c) <= 16 * U * c and float(lo) == float(hi)
    del p, g, m, v
    rows, width = 2 ** 21 + 5, 1040
    x = torch.zeros(rows, width, dtype=BF16, device=DEV)
    x[:] = randn(gen(14), 1, width, dtype=BF16)
    x[-1] = randn(gen(15), width, dtype=BF16)
    w = torch.ones(width, dtype=BF16, device=DEV)
    y, mean, rstd = torch.ops.fsctep.layer_norm(x, w, None, EPS, 0, True)
    small = x[-3:].contiguous()
    y3, mean3, rstd3 = torch.ops.fsctep.layer_norm(small, w, None, EPS, 0, True)
    assert torch.equal(y[-3:], y3) and torch.equal(mean[-3:], mean3) and torch.equal(y[0], y[rows // 2])
    dx, _, _ = torch.ops.fsctep.layer_norm_backward(x, x, w, None, mean, rstd, EPS, 0, True, False, False)
    d3, _, _ = torch.ops.fsctep.layer_norm_backward(small, small, w, None, mean3, rstd3, EPS, 0, True, False, False)
    assert torch.equal(dx[-3:], d3)
    del y
    gx, gdy, _, _ = torch.ops.fsctep.layer_norm_backward_twice(x, None, None, x, x, w, None, mean, rstd, EPS, 0, True, True, False, False)
    g3, h3, _, _ = torch.ops.fsctep.layer_norm_backward_twice(small, None, None, small, small, w, None, mean3, rstd3, EPS, 0, True,
                                                              True, False, False)
    assert torch.equal(gx[-3:], g3) and torch.equal(gdy[-3:], h3)


# ------------------------------------------------------------------ streams and graphs
def test_another_stream():
    a = norm_inputs(300, 640, F32, F32)
    t, index = torch.randn(50, 64, device=DEV, requires_grad=True), torch.randint(0, 50, (9000,), device=DEV)
    want = norm_call(silu=True, **a), torch.autograd.grad(L.embedding(t, index).sum(), t)[0]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = norm_call(silu=True, **a), torch.autograd.grad(L.embedding(t, index).sum(), t)[0]
    side.synchronize()
    assert all(torch.equal(want[0][k], got[0][k]) for k in got[0]) and torch.equal(want[1], got[1])


def capture(call):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    return graph, out


def test_captured_norm_and_lookup():
    a = norm_inputs(200, 331, F32, F32)
    table, index = torch.randn(40, 64, device=DEV), torch.randint(0, 40, (6000,), device=DEV)
    dy = torch.randn(6000, 64, device=DEV)

    def call():
        y, mean, rstd = torch.ops.fsctep.layer_norm(a["x"], a["w"], a["b"], EPS, 1, True)
        first = torch.ops.fsctep.layer_norm_backward(a["dy"], a["x"], a["w"], a["b"], mean, rstd, EPS, 1, True, True, True)
        second = torch.ops.fsctep.layer_norm_backward_twice(a["v"], None, None, a["dy"], a["x"], a["w"], a["b"], mean, rstd,
                                                            EPS, 1, True, True, True, True)
        rows = torch.ops.fsctep.embedding(table, index, 2.0)
        return [y, *first, *second, rows, torch.ops.fsctep.embedding_backward(dy, index, 40, 2.0)]

    graph, out = capture(call)
    for k in range(3):
        a["x"].mul_(1.5)
        table.add_(1.0)
        index.copy_(torch.randint(0, 40, (6000,), device=DEV))
        want = [t.clone() for t in call()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want)), k


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step(bits):
    """Replays count the steps on, and take a new learning rate and new gradients."""
    g = gen(13)
    lr = torch.full((), 1e-2, device=DEV)
    ps = [torch.nn.Parameter(randn(g, 500)), torch.nn.Parameter(randn(g, 30).to(BF16))]
    for p in ps:
        p.grad = torch.zeros_like(p)
    opt = optim.AdamW(ps, lr=lr, max_norm=1.0, state_bits=bits)
    graph, _ = capture(opt.step)
    twin = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    other = optim.AdamW(twin, lr=lr, max_norm=1.0, state_bits=bits)
    other.load_state_dict(opt.state_dict())
    other.param_groups[0]["lr"] = lr
    for k in range(4):
        lr.fill_(1e-2 / (k + 1))
        for p, q in zip(ps, twin):
            p.grad.copy_(randn(g, *p.shape))
            q.grad = p.grad.clone()
        graph.replay()
        other.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, twin)), k
        assert all(float(opt.state[p]["step"]) == float(other.state[q]["step"]) for p, q in zip(ps, twin))
