"""Steps of optim.AdamW from checkpoints, on the GPU."""

import pytest
import torch

from fsctep_amd import optim

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def test_a_step_from_torchs_states_of_16_bits():
    """A bfloat16 parameter's moments come in bfloat16; the step is AdamW's in 64 bits from the values that those stand for:
    m, v and the 32-bit copy in at most 16 roundings of their terms."""
    g = torch.Generator(device=DEV).manual_seed(1)
    p = torch.randn(300, generator=g, device=DEV).bfloat16().requires_grad_(True)
    theirs = torch.optim.AdamW([p], lr=1e-2, weight_decay=0.1)
    for _ in range(3):
        p.grad = torch.randn(300, generator=g, device=DEV).bfloat16()
        theirs.step()
    q = p.detach().clone().requires_grad_(True)
    opt = optim.AdamW([q], lr=0.5)
    opt.load_state_dict(theirs.state_dict())
    assert float(opt.state[q]["step"]) == 3
    q.grad = torch.randn(300, generator=g, device=DEV).bfloat16()
    twin = p.detach().double().requires_grad_(True)
    exact = torch.optim.AdamW([twin], lr=1e-2, weight_decay=0.1)
    exact.load_state_dict(theirs.state_dict())
    twin.grad = q.grad.double()
    opt.step()
    exact.step()
    s, t = opt.state[q], exact.state[twin]
    size = theirs.state[p]["exp_avg"].double().abs() + q.grad.double().abs()
    assert ((s["exp_avg"].double() - t["exp_avg"]).abs() <= 16 * U * size).all()
    assert ((s["exp_avg_sq"].double() - t["exp_avg_sq"]).abs() <= 16 * U * t["exp_avg_sq"]).all()
    # a step is at most a few lr, its quotient off by as many roundings
    assert ((s["master"].double() - twin.detach()).abs() <= 16 * U * (p.detach().double().abs() + 20 * 1e-2)).all()
    assert torch.equal(q.detach(), s["master"].bfloat16())
