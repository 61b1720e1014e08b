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
