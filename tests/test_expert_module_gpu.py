"""The expert readout module in bfloat16 and on the trunks.  Bounds: each value held in bfloat16 is off by at most 2^-8 of it; a
layer rounds its rows, hidden values and output, its gradient as many: 2^-6 of the largest value for a stack of two."""

import pytest
import torch

from oracle import experts as O
from sparse_helpers import rel_inf
from test_expert_readout_gpu import DEV, _attach, _system, oracle, readout

pytestmark = pytest.mark.gpu


def bf16_readout(width, hidden, experts, seed, **kw):
    return readout(width, hidden, experts, seed, **kw).bfloat16()


@pytest.mark.parametrize("rows", [5, 40, 700])
@pytest.mark.parametrize("rows_type", ["fp32", "bf16"])
@pytest.mark.parametrize("differentiable", [False, True])
def test_module_in_bf16_matches_oracle(rows, rows_type, differentiable):
    """Experts chosen by species; rows in float32 (a trunk's) and in bfloat16; all gradients."""
    m = bf16_readout(200, 72, 6, rows, k=2, layers=2, n_species=7)
    dt = torch.float32 if rows_type == "fp32" else torch.bfloat16
    g = torch.Generator().manual_seed(rows)
    x, dy = torch.randn(rows, 200, generator=g).to(dt), torch.randn(rows, 200, generator=g).to(dt)
    species = torch.randint(0, 7, (rows,), generator=g)
    leaf = x.double().requires_grad_(True)
    y0 = oracle(m, leaf, species)
    dx0, = torch.autograd.grad(y0, leaf, dy.double())
    xd = x.to(DEV).requires_grad_(True)
    y = m(xd, species.to(DEV), differentiable=differentiable)
    got = torch.autograd.grad(y, [xd, *m.parameters()], dy.to(DEV))
    assert y.dtype == dt and got[0].dtype == dt and all(t.dtype == torch.bfloat16 for t in got[1:])
    assert rel_inf(y.float(), y0) < 2.0 ** -6 and rel_inf(got[0].float(), dx0) < 2.0 ** -6
    assert all(torch.isfinite(t).all() and float(t.abs().max()) > 0 for t in got[1:])


def test_module_in_bf16_chooses_by_rows():
    m = bf16_readout(96, 40, 6, 2, k=2)
    x = torch.randn(64, 96, device=DEV)
    y = m(x)
    assert y.dtype == torch.float32 and torch.isfinite(y).all()
    assert rel_inf(m(x, differentiable=True), y) < 2.0 ** -6          # the same choice, the same roundings


def test_float32_module_takes_bf16_rows():
    m = readout(96, 40, 6, 2, k=2, layers=2, n_species=5)
    x, species = torch.randn(64, 96, device=DEV).bfloat16(), torch.arange(64, device=DEV) % 5
    y = m(x, species)
    assert y.dtype == torch.bfloat16 and rel_inf(y.float(), oracle(m, x.double().cpu(), species.cpu())) < 2.0 ** -8


def test_trunk_with_experts_in_bf16():
    """Energies and forces, the force-loss step and its parameter gradients, HIP-graph replay: the experts' contribution
    within 2^-6 of the float32 experts' with the same (rounded) parameters, a new readout's exactly zero."""
    from fsctep_amd.capture import CapturedEnergyForces
    from fsctep_amd.experts import ExpertReadout
    from fsctep_amd.sparse import energy_and_forces
    g, model, pos, A, batch, cell, (src, dst, sh) = _system()
    graph = model.prepare(src, dst, sh, pos.shape[0], A)
    e0, f0 = energy_and_forces(model, pos, batch, cell, graph)
    width = model.proj_total.input_norm.normalized_shape[0]
    model.readout_experts = ExpertReadout(width, 48, 4, n_species=model.n_species).to(DEV).bfloat16()
    e, f = energy_and_forces(model, pos, batch, cell, graph)
    assert torch.equal(e, e0) and torch.equal(f, f0)
    _attach(model, layers=2)
    model.readout_experts.bfloat16().float()
    e32, f32 = energy_and_forces(model, pos, batch, cell, graph)
    model.readout_experts.bfloat16()
    e, f = energy_and_forces(model, pos, batch, cell, graph)
    assert float((e - e32).norm()) < 2.0 ** -6 * float((e32 - e0).norm())
    assert float((f - f32).norm()) < 2.0 ** -6 * float((f32 - f0).norm())
    cap = CapturedEnergyForces(model, pos, batch, cell, graph)
    for k in range(3):
        q = pos + 0.01 * k
        ce, cf, _ = cap(q)
        ee, ef = energy_and_forces(model, q, batch, cell, graph)
        torch.cuda.synchronize()
        assert torch.equal(ce.squeeze(), ee) and torch.equal(cf, ef), k
    model.train().requires_grad_(True)
    p = pos.clone().requires_grad_(True)
    et = model(p, A, batch, src, dst, sh, cell)
    gp, = torch.autograd.grad(et.sum(), p, create_graph=True)
    assert float((gp + f).detach().norm()) < 2.0 ** -6 * float((f32 - f0).norm()) + 2e-5 * float(f0.norm())
    grads = torch.autograd.grad((gp ** 2).sum(), list(model.readout_experts.parameters()))
    assert all(t.dtype == torch.bfloat16 and torch.isfinite(t).all() and float(t.abs().max()) > 0 for t in grads)


@pytest.mark.parametrize("differentiable", [False, True])
def test_atoms_without_a_row_become_nan(differentiable):
    """Atomic numbers outside the table, and only they."""
    m = readout(96, 40, 6, 2, k=2, layers=2, n_species=5)
    x = torch.randn(64, 96, device=DEV)
    species = torch.arange(64, device=DEV) % 5
    want = m(x, species, differentiable=differentiable)
    for other in (5, -1, 2 ** 40):
        bad = species.clone()
        bad[7] = other
        y = m(x, bad, differentiable=differentiable)
        assert torch.isnan(y[7]).all()
        y[7] = want[7]
        assert rel_inf(y, want) < 2e-5
    assert torch.isnan(m.to_8_bits()(x, bad)[7]).all()


def test_a_trunk_with_experts_that_know_fewer_elements():
    """Its own elements as with a table of all; an atom of an element beyond the table NaN, no other atom's."""
    g, model, pos, A, batch, cell, (src, dst, sh) = _system()
    graph = model.prepare(src, dst, sh, pos.shape[0], A)
    _attach(model)
    with torch.no_grad():
        e0 = model.forward_graph(pos, batch, cell, graph)
        for known in (int(A.max()) + 1, int(A.max())):
            full = model.readout_experts
            few = readout(model.proj_total.input_norm.normalized_shape[0], 48, 4, 3, n_species=known)
            few.load_state_dict({k: v[:known] if k.endswith("gate") else v for k, v in full.state_dict().items()})
            model.readout_experts = few
            e = model.forward_graph(pos, batch, cell, graph)
            model.readout_experts = full
            has = A < known
            assert torch.equal(e[has], e0[has]) and torch.isnan(e[~has]).all()
    assert not has.all() and has.any()


@pytest.mark.parametrize("kw", [dict(k=2, layers=2, score="sigmoid", n_species=7), dict(k=2, layers=1),
                                dict(k=1, layers=2, renormalise=False, scale=2.0, n_species=7)])
def test_parameter_gradients_of_a_force_loss(kw):
    """The gradient of sum (d(m(x) . dy)/dx)^2 with respect to every parameter, against 64 bits (1e-4 of the largest value:
    two derivatives of fp32 sums of 130 x 96 products, 1e-6 of each term)."""
    m = readout(96, 40, 6, 1, **kw)
    g = torch.Generator().manual_seed(4)
    x, dy = torch.randn(130, 96, generator=g), torch.randn(130, 96, generator=g)
    species = torch.randint(0, 7, (130,), generator=g) if kw.get("n_species") else None
    p0 = [{n: p.detach().double().cpu().requires_grad_(True) for n, p in layer.named_parameters()} for layer in m.layers]
    leaf, r = x.double().requires_grad_(True), m.router
    out = leaf
    for p, layer in zip(p0, m.layers):
        y, _ = O.rms_norm(out, p["norm"], eps=m.eps)
        logits = y @ p["gate"].T if species is None else p["gate"][species]
        index = O.choose(O.scores(logits.detach(), r.score) + layer.balance.double().cpu(), r.k)
        out = out + O.expert_mlp(y, index, O.weights(logits, index, r.score, r.renormalise, r.scale), p["w_in"], p["w_out"])
    f0, = torch.autograd.grad((out * dy.double()).sum(), leaf, create_graph=True)
    ref = torch.autograd.grad((f0 ** 2).sum(), [p[n] for p in p0 for n in p], allow_unused=True)
    xd = x.to(DEV).requires_grad_(True)
    y = m(xd, None if species is None else species.to(DEV), differentiable=True)
    f, = torch.autograd.grad((y * dy.to(DEV)).sum(), xd, create_graph=True)
    got = torch.autograd.grad((f ** 2).sum(), [q for layer in m.layers for q in layer.parameters()], allow_unused=True)
    assert rel_inf(f.detach(), f0.detach()) < 1e-5
    names = [n for layer in m.layers for n, _ in layer.named_parameters()]
    assert names == [n for p in p0 for n in p]
    for n, a, b in zip(names, got, ref):
        assert (a is None) == (b is None) and (a is None or rel_inf(a, b) < 1e-4), n


def test_trunk_energies_in_8_bits_are_near():
    """The energies' change by 8-bit experts, against what the experts change: their outputs are within 5 %, the head's
    response to an error that of any direction, four times that at most."""
    g, model, pos, A, batch, cell, (src, dst, sh) = _system()
    graph = model.prepare(src, dst, sh, pos.shape[0], A)
    with torch.no_grad():
        e0 = model.forward_graph(pos, batch, cell, graph)
        _attach(model, layers=2)
        e = model.forward_graph(pos, batch, cell, graph)
        model.readout_experts = model.readout_experts.to_8_bits()
        e8 = model.forward_graph(pos, batch, cell, graph)
    assert float((e8 - e).norm()) < 0.2 * float((e - e0).norm())


def test_ictd_forces_with_experts():
    """The fused path's energies and forces against the twice differentiable torch form of the training step, and against
    differences of the energy."""
    from conftest import load_golden
    from fsctep_amd.ictd import energy_forces
    from test_ictd_gpu import _model
    g = load_golden("ictd_open32_c32_l2")
    model = _attach(_model(g))
    t = lambda k, dt=None: torch.tensor(g[k], device=DEV, dtype=dt)
    pos, A, cell = t("pos", torch.float32), t("species"), t("cell", torch.float32)
    batch = torch.zeros(pos.shape[0], dtype=torch.long, device=DEV)
    src, dst, sh = t("edge_src"), t("edge_dst"), t("edge_shifts", torch.float32)
    graph = model.prepare(src, dst, sh, pos.shape[0], A)
    e, f, _ = energy_forces(model, pos, batch, cell, graph)
    h, d = 1e-2, torch.randn(pos.shape, generator=torch.Generator().manual_seed(2)).to(DEV)
    sums = [float(energy_forces(model, pos + s * h * d, batch, cell, graph)[0].double().sum()) for s in (2, 1, -1, -2)]
    slope = (-sums[0] + 8 * sums[1] - 8 * sums[2] + sums[3]) / (12 * h)
    assert abs(slope + float((f.double() * d.double()).sum())) < 2e-2 * float(f.double().norm() * d.double().norm())
    model.train().requires_grad_(True)
    p = pos.clone().requires_grad_(True)
    et = model(p, A, batch, src, dst, sh, cell)
    et = et[0] if isinstance(et, tuple) else et
    gp, = torch.autograd.grad(et.sum(), p, create_graph=True)
    assert rel_inf(et.detach().squeeze(-1), e.squeeze(-1) if e.dim() > 1 else e) < 2e-5 and rel_inf(-gp.detach(), f) < 2e-5
    grads = torch.autograd.grad((gp ** 2).sum(), list(model.readout_experts.parameters()))
    assert all(torch.isfinite(q).all() and float(q.abs().max()) > 0 for q in grads)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("scale", [1.0, 1.5, 0.3, 2.7])
def test_a_single_renormalised_choice_has_no_gradient(score, scale):
    """Its weight is the scale whatever the logits: zero to the bit."""
    from fsctep_amd import expert_ops as X
    for experts in (1, 7, 40):
        l = torch.randn(500, experts, device=DEV, requires_grad=True)
        index, w = X.route_experts(l, 1, score=score, scale=scale)
        dl, = torch.autograd.grad(w, l, torch.randn(500, 1, device=DEV))
        assert torch.equal(w, torch.full_like(w, scale)) and float(dl.abs().max()) == 0
