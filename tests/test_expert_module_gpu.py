"""The expert readout module in bfloat16 and on the trunks.  Bounds: each value held in bfloat16 is off by at most 2^-8 of it; a
layer rounds its rows, hidden values and output, its gradient as many: 2^-6 of the largest value for a stack of two."""

import pytest
import torch

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
