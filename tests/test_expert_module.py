"""The expert readout module and its twice differentiable forms on the CPU (the fused operators run on the GPU only)."""

import math

import pytest
import torch

from fsctep_amd import train_ops as T
from fsctep_amd.experts import ExpertReadout
from oracle import experts as O


def test_the_balance_bias_stays_float32():
    """The router takes a float32 bias; casting the parameters leaves it, whatever its values."""
    m = ExpertReadout(20, 8, 4, k=2)
    with torch.no_grad():
        m.layers[0].balance.copy_(torch.tensor([0.1, -0.2, 1e-3, 0.0]))
    want = m.layers[0].balance.clone()
    for cast in (lambda: m.bfloat16(), lambda: m.to(torch.bfloat16), lambda: m.float()):
        cast()
        assert m.layers[0].balance.dtype == torch.float32 and torch.equal(m.layers[0].balance, want)
    assert m.bfloat16().layers[0].w_in.dtype == torch.bfloat16
    m.layers[0].rebalance(torch.zeros(1000, 1, dtype=torch.int32), rate=0.5)   # counts of more than bfloat16 holds
    assert torch.equal(m.layers[0].balance, want + torch.tensor([-0.5, 0.5, 0.5, 0.5]))
    eight = m.to_8_bits().bfloat16()
    assert all(b.dtype in (torch.float32, torch.int8) for b in eight.buffers())
    assert m.to("meta").layers[0].balance.dtype == torch.float32


def test_rows_of_other_types_are_refused():
    m = ExpertReadout(20, 8, 4)
    for differentiable in (False, True):
        with pytest.raises(ValueError, match="float32 or bfloat16"):
            m(torch.zeros(3, 20, dtype=torch.float64), differentiable=differentiable)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_twice_differentiable_forms_sum_in_32_bits(score):
    """bfloat16 operands, one rounding: the norm's values are the 64-bit ones rounded (a neighbour where 32 bits fall on the
    other side of a half), the products' within 2^-8 of the largest."""
    g = torch.Generator().manual_seed(3)
    rn = lambda *s: torch.randn(*s, generator=g)
    x, w = rn(50, 640).bfloat16(), (1 + 0.3 * rn(640)).bfloat16()
    y, _ = T.rms_norm(x, w)
    y0, _ = O.rms_norm(x, w)
    assert y.dtype == torch.bfloat16 and float((y == y0.bfloat16()).double().mean()) > 0.999
    logits = rn(50, 6).bfloat16()
    index = O.choose(O.scores(logits, score), 2)
    weight = T.route_weights(logits, index, score, True, 1.0)
    assert weight.dtype == torch.float32 and torch.allclose(weight.double(), O.weights(logits, index, score), rtol=1e-6, atol=0)
    w_in, w_out = (rn(6, 80, 640) / math.sqrt(640)).bfloat16(), (rn(6, 640, 40) / math.sqrt(40)).bfloat16()
    y = T.expert_mlp(x, index, weight, w_in, w_out)
    y0 = O.expert_mlp(x, index, weight, w_in, w_out)
    assert y.dtype == torch.bfloat16 and float((y.double() - y0).abs().max()) <= 2.0 ** -8 * float(y0.abs().max())


def test_an_index_outside_the_experts_adds_nothing():
    """As the fused operator has it: below 0 and from n_experts on."""
    g = torch.Generator().manual_seed(5)
    rn = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    x, w_in, w_out, weight = rn(4, 12), rn(3, 10, 12), rn(3, 12, 5), torch.rand(4, 2, generator=g, dtype=torch.float64)
    index = torch.tensor([[0, 3], [7, 2], [-1, 2 ** 30], [1, -9]], dtype=torch.int32)
    x.requires_grad_(True)
    y, y0 = T.expert_mlp(x, index, weight, w_in, w_out), O.expert_mlp(x, index, weight, w_in, w_out)
    assert torch.allclose(y, y0, rtol=1e-12, atol=1e-14) and float(y[2].detach().abs().max()) == 0
    logits = rn(4, 3).requires_grad_(True)
    picked = T.route_weights(logits, index, "softmax", False, 2.0)
    want = torch.where((index >= 0) & (index < 3), 2 * torch.softmax(logits, -1).gather(1, index.clamp(0, 2).long()), 0.0)
    assert torch.allclose(picked, want, rtol=1e-12, atol=0)
    layer = ExpertReadout(20, 8, 4).layers[0]
    layer.rebalance(torch.tensor([[0, 4], [9, -1], [0, 2]], dtype=torch.int32), rate=0.5)    # counts 2, 0, 1, 0
    assert layer.balance.tolist() == [-0.5, 0.5, -0.5, 0.5]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [False, True])
def test_rows_with_nothing_to_choose_have_no_gradient(score, renormalise):
    """A row whose logits are all -inf (and one barred in part) beside ordinary rows: zeros, and so through the second
    derivative; the other rows' gradient is the formula's."""
    g = torch.Generator().manual_seed(6)
    logits = torch.randn(4, 5, generator=g, dtype=torch.float64)
    logits[1] = -math.inf
    logits[2, :3] = -math.inf
    index = O.choose(torch.where(logits > -math.inf, O.scores(logits, score), -math.inf), 2)   # a barred expert is not chosen
    assert index[1].tolist() == [-1, -1]
    u = torch.randn(4, 2, generator=g, dtype=torch.float64)
    leaf = logits.clone().requires_grad_(True)
    w = T.route_weights(leaf, index, score, renormalise, 1.5)
    dl, = torch.autograd.grad((w * u).sum(), leaf, create_graph=True)
    second, = torch.autograd.grad((dl ** 2).sum(), leaf)
    assert float(w[1].detach().abs().max()) == 0 and float(dl[1].detach().abs().max()) == 0
    assert torch.isfinite(second).all() and float(second[1].abs().max()) == 0
    want = O.route_gradient(logits, index, score, renormalise, 1.5, u)
    assert torch.allclose(dl, want, rtol=1e-12, atol=1e-14)


def test_atomic_numbers_without_a_row():
    """Looked up nowhere: NaN logits, unless the caller's bound lies within the table."""
    r = ExpertReadout(20, 8, 4, n_species=5)
    layer = r.layers[0]
    species = torch.tensor([0, 4, 5, -1, 2 ** 40, 3])
    l = r.router.logits(layer, None, *r.router.rows_of(species, None))
    ok = torch.tensor([True, True, False, False, False, True])
    assert torch.equal(l[ok], layer.gate.detach()[species[ok]]) and torch.isnan(l[~ok]).all()
    g, = torch.autograd.grad(l[ok].sum(), layer.gate)
    assert torch.isfinite(g).all()
    assert torch.equal(r.router.logits(layer, None, *r.router.rows_of(species[ok], 5)), l[ok])
    assert r.router.rows_of(species[ok], 5)[1] is None and r.router.rows_of(species[ok], 4)[1] is None
    l = r.router.logits(layer, None, *r.router.rows_of(species, 100))       # a bound beyond the table: looked at
    assert torch.isnan(l[~ok]).all() and torch.isfinite(l[ok]).all()
    for m in (r, r.to_8_bits()):
        with pytest.raises(ValueError, match="pass species"):
            m(torch.zeros(6, 20))


def test_codes_of_the_smallest_numbers_keep_their_sign():
    from fsctep_amd.expert_ops import to_codes
    w = torch.tensor([[190.0, 3.0, -190.0], [127.0, 1.0, -2.0], [0.0, 0.0, 0.0]]) * 2.0 ** -149
    q, s = to_codes(w)
    assert q.tolist() == [[127, 3, -127], [127, 1, -2], [0, 0, 0]]
    q, s = to_codes(w * 2.0 ** 120)
    assert q.tolist() == [[127, 2, -127], [127, 1, -2], [0, 0, 0]]
    assert float((q * s.unsqueeze(1) - w * 2.0 ** 120).abs().max()) <= 0.5 * float(s.max())


def test_twice_differentiable_products_keep_what_nobody_asks_for_out():
    """NaN and infinities in an expert that nobody chose and in a row without an expert: not in the products, not in any
    gradient of theirs, first or second."""
    g = torch.Generator().manual_seed(8)
    rn = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    x, w_in, w_out, weight = rn(5, 12), rn(3, 10, 12), rn(3, 12, 5), torch.rand(5, 2, generator=g, dtype=torch.float64)
    index = torch.tensor([[0, 2], [2, -1], [-1, 3], [0, 0], [2, 0]], dtype=torch.int32)
    dy = rn(5, 12)
    leaf0 = [t.clone().requires_grad_(True) for t in (x, weight, w_in, w_out)]
    y0 = O.expert_mlp(leaf0[0], index, *leaf0[1:])
    first0 = torch.autograd.grad((y0 * dy).sum(), leaf0, create_graph=True)
    second0 = torch.autograd.grad((first0[0] ** 2).sum(), leaf0)
    x[2], w_in[1], w_out[1], weight[2, 0] = math.nan, math.inf, math.nan, math.nan
    leaf = [t.clone().requires_grad_(True) for t in (x, weight, w_in, w_out)]
    y = T.expert_mlp(leaf[0], index, *leaf[1:])
    first = torch.autograd.grad((y * dy).sum(), leaf, create_graph=True)
    second = torch.autograd.grad((first[0] ** 2).sum(), leaf)
    for a, b in zip((y, *first, *second), (y0, *first0, *second0)):
        assert torch.allclose(a, b, rtol=1e-11, atol=1e-13)
