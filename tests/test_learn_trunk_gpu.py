"""The training step's operators where the trunks and the expert readout call them, and a run of them together: steps of
force training with the optimiser against the fp64 oracle and torch's AdamW in 64 bits."""

import numpy as np
import pytest
import torch
import torch.nn as nn

from conftest import load_golden
from fsctep_amd import learn_ops, optim, train_ops as T
from fsctep_amd.experts import ExpertReadout

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def system(g):
    n = g["pos"].shape[0]
    return (torch.zeros(n, dtype=torch.long, device=DEV), torch.tensor(g["cell"], dtype=torch.float32, device=DEV),
            torch.tensor(g["edge_src"], device=DEV), torch.tensor(g["edge_dst"], device=DEV),
            torch.tensor(g["edge_shifts"], dtype=torch.float32, device=DEV), torch.tensor(g["species"], device=DEV))


def oracle_steps(energy, params, pos, e_ref, f_ref, steps, **rule):
    """The parameters after each of the steps, and each step's loss, in 64 bits on the CPU."""
    p = {k: v.clone().requires_grad_(True) for k, v in params.items()}
    opt = torch.optim.AdamW(list(p.values()), **rule)
    losses, largest = [], 0.0
    for _ in range(steps):
        x = pos.clone().requires_grad_(True)
        e = energy(x, p)
        gx, = torch.autograd.grad(e.sum(), x, create_graph=True)
        loss = 1.0 * (e.sum() - e_ref).square() + 10.0 * (gx + f_ref).square().mean()
        grads = torch.autograd.grad(loss, list(p.values()), allow_unused=True)
        for t, g in zip(p.values(), grads):
            t.grad = g
        largest = max(largest, max(float(g.abs().max()) for g in grads if g is not None))
        opt.step()
        losses.append(float(loss))
    return {k: v.detach() for k, v in p.items()}, losses, largest


def run_steps(m, g, ref_energy, params, steps=3):
    """A step's gradients are within 2e-5 of the largest one of all (tests/test_trunk_train_gpu.py holds each parameter's to that
    of its own); with eps at a tenth of the largest, m / (sqrt(v) + eps) is off by at most twice that over eps a step: 4e-4 lr,
    steps add, and the parameters' own roundings, 8 a step."""
    n = g["pos"].shape[0]
    batch, cell, src, dst, sh, A = system(g)
    pos = torch.tensor(g["pos"], dtype=torch.float32, device=DEV)
    rng = np.random.default_rng(3)
    f_ref = torch.tensor(rng.normal(size=(n, 3)), dtype=torch.float32)
    e_ref = torch.tensor([float(np.sum(g["energy_f64"])) + 0.3], dtype=torch.float32)
    lr = 1e-4
    rule = dict(lr=lr, betas=(0.9, 0.99), weight_decay=0.01)
    _, _, largest = oracle_steps(ref_energy, params, pos.double().cpu(), e_ref.double(), f_ref.double(), 1, eps=1.0, **rule)
    eps = largest / 10
    want, losses, _ = oracle_steps(ref_energy, params, pos.double().cpu(), e_ref.double(), f_ref.double(), steps, eps=eps, **rule)
    m.train().requires_grad_(True)
    graph = m.prepare(src, dst, sh, n, A)
    opt = optim.AdamW(m.parameters(), eps=eps, **rule)
    for k in range(steps):
        loss, e, f = optim.train_step(m, opt, pos, batch, cell, graph, e_ref.to(DEV), f_ref.to(DEV), 1.0, 10.0)
        assert e.shape == (1,) and f.shape == (n, 3)
        # energies and forces to 1e-5 of their largest: the squares' sum to a few times that
        assert abs(float(loss) - losses[k]) <= 1e-4 * losses[k]
    got = dict(m.named_parameters())
    assert set(got) == set(want)
    for name, p in got.items():
        off = (p.detach().double().cpu() - want[name]).abs().max()
        assert float(off) <= steps * (4e-4 * lr + 8 * U * float(want[name].abs().max())), name
        if p.grad is not None and float(p.grad.abs().max()) > 0:
            assert p in opt.state


def test_sparse_training_steps():
    from oracle import sparse_ref as R
    from sparse_helpers import oracle_params, seeded_hip_model
    g = load_golden("sparse_open32_c32_l2")
    C, layers, seed = int(g["channels"]), int(g["layers"]), int(g["param_seed"])
    cfg, p = oracle_params(C, layers, seed, torch.float64)
    n = g["pos"].shape[0]
    args = (torch.tensor(g["species"]), torch.zeros(n, dtype=torch.long), torch.tensor(g["edge_src"]),
            torch.tensor(g["edge_dst"]), torch.tensor(g["edge_shifts"], dtype=torch.float32).double(),
            torch.tensor(g["cell"], dtype=torch.float32).double())
    run_steps(seeded_hip_model(C, layers, seed).to(DEV), g, lambda x, prm: R.atom_energies(x, *args, prm, cfg), p)


def test_ictd_training_steps():
    from fsctep_amd.synthetic import seeded_value
    from oracle import ictd_ref as I
    from test_ictd_gpu import _model
    g = load_golden("ictd_open32_c32_l2")
    cfg = I.ICTDConfig(channels=int(g["channels"]), lmax=int(g["lmax"]), num_interaction=int(g["layers"]),
                       function_type=str(g["function_type"]), o3=False, active=(), external_field=False, dipole=False)
    p = {k: torch.tensor(seeded_value(k, s, int(g["param_seed"])), dtype=torch.float64) for k, s in I.param_shapes(cfg)}
    n = g["pos"].shape[0]
    args = (torch.tensor(g["species"]), torch.zeros(n, dtype=torch.long), torch.tensor(g["edge_src"]),
            torch.tensor(g["edge_dst"]), torch.tensor(g["edge_shifts"], dtype=torch.float32).double(),
            torch.tensor(g["cell"], dtype=torch.float32).double())
    run_steps(_model(g), g, lambda x, prm: I.forward(x, *args, prm, cfg, None)[0], p)


def head(width=224):
    from fsctep_amd.sparse import MainNet, RobustScalarWeightedSum
    torch.manual_seed(2)
    net, ws = MainNet(width, [128, 128, 128], 17), RobustScalarWeightedSum(17, "random")
    with torch.no_grad():
        for ln in (net.input_norm, *net.layer_norms):
            ln.weight.add_(0.2 * torch.randn_like(ln.weight))
            ln.bias.add_(0.2 * torch.randn_like(ln.bias))
        net.output.weight.mul_(20)
    return net.to(DEV), ws.to(DEV)


def head_grads(call, net, ws, x, v):
    """The energies, their gradient, and the gradients of (dx . v)^2 with respect to rows and parameters."""
    x = x.detach().requires_grad_(True)
    e = call(net, ws, x)
    dx, = torch.autograd.grad(e.sum(), x, create_graph=True)
    ps = [*net.parameters(), *ws.parameters()]
    return [e, dx, *torch.autograd.grad(((dx * v).sum(1) ** 2).sum() + (e ** 2).sum(), [x, *ps], allow_unused=True)]


def test_the_head_differentiates_as_the_modules_do():
    """Against the modules in 64 bits, each gradient within 2e-5 of its largest value (the bound of the trunks' gradients)."""
    net, ws = head()
    g = torch.Generator(device=DEV).manual_seed(4)
    x, v = (torch.randn(301, 224, generator=g, device=DEV) for _ in range(2))
    got = head_grads(T.readout_energy, net, ws, x, v)
    net6, ws6 = head()
    want = head_grads(lambda n, w, t: w(n(t)), net6.double(), ws6.double(), x.double(), v.double())
    names = [str(n) for n, _ in net.named_parameters()]
    floor = 1e-3 * max(float(w.abs().max()) for w in want[2:] if w is not None)
    for i, (a, b) in enumerate(zip(got, want)):
        assert (a is None) == (b is None)
        if a is not None:
            assert float((a.double() - b).abs().max()) <= 2e-5 * max(float(b.abs().max()), floor), (i, names)


def test_other_heads_run_as_the_modules(monkeypatch):
    """A hook is called, another kind of norm and 64-bit rows are taken, autocast keeps its types."""
    net, ws = head()
    x = torch.randn(7, 224, device=DEV)
    want = ws(net(x))
    calls = []
    real = learn_ops.layer_norm
    monkeypatch.setattr(learn_ops, "layer_norm", lambda *a, **k: calls.append(1) or real(*a, **k))
    assert torch.allclose(T.readout_energy(net, ws, x), want, rtol=1e-5, atol=1e-6) and len(calls) == 4
    calls.clear()
    seen = []
    hook = net.layer_norms[1].register_forward_hook(lambda *a: seen.append(1))
    assert torch.equal(T.readout_energy(net, ws, x), want) and seen and not calls
    hook.remove()
    hook = net.register_forward_hook(lambda *a: seen.append(2))
    assert torch.equal(T.readout_energy(net, ws, x), want) and seen[-1] == 2 and not calls
    hook.remove()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(T.readout_energy(net, ws, x), ws(net(x))) and not calls

    class Other(nn.LayerNorm):
        pass

    net.layer_norms[0] = Other(128).to(DEV)
    assert torch.equal(T.readout_energy(net, ws, x), ws(net(x))) and not calls
    net6, ws6 = head()
    net6, ws6 = net6.double(), ws6.double()
    assert torch.equal(T.readout_energy(net6, ws6, x.double()), ws6(net6(x.double()))) and not calls


@pytest.mark.parametrize("shape", [(9, 5), (9, 3, 4), (4,)])
def test_lookup_of_tables(shape):
    g = torch.Generator(device=DEV).manual_seed(6)
    t = torch.randn(*shape, generator=g, device=DEV, requires_grad=True)
    index = torch.randint(0, shape[0], (2000,), generator=g, device=DEV, dtype=torch.int32)
    if t.dim() == 1:
        t = t.detach().unsqueeze(1).requires_grad_(True)
    y = T.lookup(t, index)
    assert torch.equal(y, t.index_select(0, index.long()))
    dy = torch.randn(y.shape, generator=g, device=DEV)
    got, = torch.autograd.grad(y, t, dy)
    want = torch.zeros(t.shape, dtype=torch.float64, device=DEV).index_add_(0, index.long(), dy.double())
    size = torch.zeros(t.shape, dtype=torch.float64, device=DEV).index_add_(0, index.long(), dy.double().abs())
    assert ((got.double() - want).abs() <= 2000 * U * size).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_expert_scores_by_atomic_number(dtype):
    """The table's gradient through the expert readout, in both of its forms, against autograd in 64 bits on the table's own
    lookup: a sum of the atoms' rows, rounded once."""
    torch.manual_seed(7)
    m = ExpertReadout(64, 32, 4, k=2, n_species=10).to(DEV, dtype)
    with torch.no_grad():
        m.layers[0].w_out.normal_(0, 0.1)
    species = torch.randint(0, 10, (500,), device=DEV)
    gate = m.layers[0].gate
    rows = m.router.logits(m.layers[0], None, species)
    assert torch.equal(rows, gate.index_select(0, species))
    dy = torch.randn(rows.shape, device=DEV).to(dtype)
    got, = torch.autograd.grad(rows, gate, dy)
    want = torch.zeros(gate.shape, dtype=torch.float64, device=DEV).index_add_(0, species, dy.double())
    size = torch.zeros(gate.shape, dtype=torch.float64, device=DEV).index_add_(0, species, dy.double().abs())
    tol = 500 * U * size + (2.0 ** -8 * want.abs() if dtype == torch.bfloat16 else 0)
    assert ((got.double() - want).abs() <= tol).all()
    x = torch.randn(500, 64, device=DEV, dtype=dtype)
    for differentiable in (False, True):
        g2, = torch.autograd.grad(m(x, species, differentiable=differentiable, species_below=10).float().square().sum(), gate)
        assert torch.isfinite(g2).all() and float(g2.float().abs().sum()) > 0


def test_training_in_bfloat16_with_copies():
    """An expert layer in bfloat16: its steps follow the 32-bit copies, also where a step is below the parameter's own."""
    torch.manual_seed(8)
    m = ExpertReadout(64, 32, 4, k=2, n_species=10).to(DEV).bfloat16()
    with torch.no_grad():
        m.layers[0].w_out.normal_(0, 0.1)
    x, species = torch.randn(200, 64, device=DEV, dtype=torch.bfloat16), torch.randint(0, 10, (200,), device=DEV)
    for bits in (32, 8):
        opt = optim.AdamW(m.parameters(), lr=1e-5, weight_decay=0.0, max_norm=1.0, state_bits=bits)
        before = {n: p.detach().float().clone() for n, p in m.named_parameters()}
        for _ in range(5):
            opt.zero_grad()
            m(x, species).float().square().mean().backward()
            opt.step()
        assert float(opt.grad_norm) > 0
        for n, p in m.named_parameters():
            s = opt.state[p]
            assert torch.equal(p, s["master"].bfloat16()) and p.dtype == torch.bfloat16
            moved = (s["master"] - before[n]).abs()
            # five steps of at most lr (1 + the quotient's own spread at 8 bits) each
            assert 0 < float(moved.max()) <= 5 * 1e-5 * 1.7
