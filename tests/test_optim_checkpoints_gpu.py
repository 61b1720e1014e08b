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


def test_a_float32_run_between_two_of_16_bits():
    """The second bfloat16 run goes on from what the float32 run left, not from the first one's copies."""
    def run(dtype, values, held, lr):
        p = values.to(dtype).requires_grad_(True)
        opt = optim.AdamW([p], lr=lr, weight_decay=0.0)
        if held is not None:
            opt.load_state_dict(held)
        for group in opt.param_groups:
            group["lr"] = lr
        p.grad = torch.ones_like(p)
        opt.step()
        return p.detach(), opt.state_dict()

    start = torch.linspace(-1, 1, 300, device=DEV)
    a, held = run(torch.bfloat16, start, None, 0.0)
    b, held = run(torch.float32, a.float() + 1.0, held, 0.0)
    c, held = run(torch.bfloat16, b, held, 0.0)
    assert torch.equal(b, a.float() + 1.0) and torch.equal(c, b.bfloat16())
    assert torch.equal(held["state"][0]["master"], c.float())


def test_values_that_come_after_the_states():
    """A program that loads the optimiser before the model, from a checkpoint without 32-bit copies."""
    q = torch.ones(300, device=DEV, requires_grad=True)
    theirs = torch.optim.AdamW([q], lr=0.0, weight_decay=0.0)
    q.grad = torch.ones_like(q)
    theirs.step()
    p = torch.zeros(300, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    opt = optim.AdamW([p], lr=0.0, weight_decay=0.0)
    opt.load_state_dict(theirs.state_dict())
    with torch.no_grad():
        p.fill_(3.0)
    p.grad = torch.ones_like(p)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="take a step before"):
        with torch.cuda.graph(graph):
            torch.zeros(1, device=DEV)
            opt.step()
    opt.step()
    assert (p == 3.0).all() and (opt.state[p]["master"] == 3.0).all() and float(opt.state[p]["step"]) == 2


def test_a_learning_rate_on_the_gpu_comes_back_from_the_host(tmp_path):
    """A checkpoint is read with its tensors on the host; the states go where the parameters are, and so does the rate."""
    p = torch.linspace(-1, 1, 300, device=DEV).requires_grad_(True)
    opt = optim.AdamW([p], lr=torch.full((), 1e-2, device=DEV))
    p.grad = torch.ones_like(p)
    opt.step()
    torch.save(opt.state_dict(), tmp_path / "opt.pt")
    q = p.detach().clone().requires_grad_(True)
    other = optim.AdamW([q], lr=0.5)
    other.load_state_dict(torch.load(tmp_path / "opt.pt", map_location="cpu", weights_only=True))
    q.grad = torch.ones_like(q)
    opt.step()
    other.step()
    assert torch.equal(p, q) and other.param_groups[0]["lr"].device == p.device


def test_a_model_that_goes_to_float32_and_back():
    """The copy of the first bfloat16 steps is not taken back after steps in float32."""
    p = torch.linspace(-1, 1, 300, device=DEV).bfloat16().requires_grad_(True)
    opt = optim.AdamW([p], lr=0.0, weight_decay=0.0)

    def step(values):
        p.data = values
        p.grad = torch.ones_like(p)
        opt.step()
        assert torch.equal(p.detach(), values) and ("master" in opt.state[p]) == (p.dtype == torch.bfloat16)

    step(p.data)
    step(p.data.float() + 1.0)
    step((p.data + 1.0).bfloat16())
    assert float(opt.state[p]["step"]) == 3 and torch.equal(opt.state[p]["master"], p.detach().float())
