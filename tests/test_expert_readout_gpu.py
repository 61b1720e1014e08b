"""The expert readout as a program uses it: the module against the 64-bit oracle, and attached to the trunks
(energies, forces, force-loss training, the traced core, HIP-graph replay, 8-bit energies).  Bounds: 1e-5 of the
largest value for fp32 values against 64 bits (2e-5 between two fp32 evaluations); the 8-bit form within 5 % of the
experts' contribution (three values held in 8 bits, 1/127 of the largest each)."""

import numpy as np
import pytest
import torch

from conftest import load_golden
from oracle import experts as O
from sparse_helpers import rel_inf, seeded_hip_model

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def readout(width, hidden, experts, seed, **kw):
    from fsctep_amd.experts import ExpertReadout
    torch.manual_seed(seed)
    m = ExpertReadout(width, hidden, experts, **kw)
    with torch.no_grad():
        for layer in m.layers:
            layer.w_out.copy_(torch.randn_like(layer.w_out) / hidden ** 0.5)
            layer.norm.copy_(1 + 0.2 * torch.randn_like(layer.norm))
            layer.balance.copy_(0.01 * torch.randn_like(layer.balance))
    return m.to(DEV)


def oracle(m, x, species=None):
    """The module in 64 bits on the CPU, choices included."""
    r = m.router
    for layer in m.layers:
        p = {k: v.detach().double().cpu() for k, v in layer.state_dict().items()}
        y, _ = O.rms_norm(x, p["norm"], eps=m.eps)
        logits = y @ p["gate"].T if species is None else p["gate"][species]
        c = O.scores(logits.detach(), r.score) + p["balance"]
        index = O.choose(c, r.k, r.groups, r.groups_kept, r.group_best)
        weight = O.weights(logits, index, r.score, r.renormalise, r.scale)
        x = x + O.expert_mlp(y, index, weight, p["w_in"], p["w_out"])
    return x


@pytest.mark.parametrize("rows,width,hidden,experts,kw", [
    (32, 640, 64, 8, dict(k=2)), (301, 200, 72, 16, dict(k=3, layers=2, score="sigmoid", groups=4, groups_kept=2, group_best=2)),
    (50, 130, 33, 5, dict(k=1, layers=3, renormalise=False, scale=2.0)),
    (70, 130, 40, 6, dict(k=2, layers=2, n_species=7))])
def test_module_matches_oracle(rows, width, hidden, experts, kw):
    m = readout(width, hidden, experts, rows, **kw)
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, width, generator=g)
    dy = torch.randn(rows, width, generator=g)
    species = torch.randint(0, 7, (rows,), generator=g) if kw.get("n_species") else None
    dev = None if species is None else species.to(DEV)
    leaf = x.double().requires_grad_(True)
    y0 = oracle(m, leaf, species)
    dx0, = torch.autograd.grad(y0, leaf, dy.double())
    xd = x.to(DEV).requires_grad_(True)
    for differentiable in (False, True):
        y = m(xd, dev, differentiable=differentiable)
        dx, = torch.autograd.grad(y, xd, dy.to(DEV))
        assert rel_inf(y, y0) < 1e-5 and rel_inf(dx, dx0) < 1e-5, differentiable


def test_module_parameter_gradients():
    m = readout(96, 40, 6, 1, k=2, layers=2, score="sigmoid")
    x = torch.randn(130, 96, device=DEV)
    dy = torch.randn(130, 96, device=DEV)
    params = [p for p in m.parameters()]
    fused = torch.autograd.grad(m(x), params, dy)
    plain = torch.autograd.grad(m(x, differentiable=True), params, dy)
    for a, b in zip(fused, plain):
        assert rel_inf(a, b) < 2e-5


def test_second_derivative_of_the_fused_form_is_refused():
    m = readout(96, 40, 6, 1)
    x = torch.randn(9, 96, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(m(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="not implemented"):
        torch.autograd.grad(g.sum(), x)


def _system():
    g = load_golden("sparse_open32_c32_l2")
    model = seeded_hip_model(int(g["channels"]), int(g["layers"]), int(g["param_seed"])).to(DEV)
    t = lambda k, **kw: torch.tensor(g[k], device=DEV, **kw)
    pos, A = t("pos", dtype=torch.float32), t("species")
    batch = torch.zeros(pos.shape[0], dtype=torch.long, device=DEV)
    cell = t("cell", dtype=torch.float32)
    args = (t("edge_src"), t("edge_dst"), t("edge_shifts", dtype=torch.float32))
    return g, model, pos, A, batch, cell, args


def _attach(model, seed=3, **kw):
    width = model.proj_total.input_norm.normalized_shape[0]
    model.readout_experts = readout(width, 48, 4, seed, n_species=model.n_species, **kw).requires_grad_(False)
    return model


def test_a_new_readout_keeps_a_trunks_energies():
    from fsctep_amd.experts import ExpertReadout
    from fsctep_amd.sparse import energy_and_forces
    g, model, pos, A, batch, cell, (src, dst, sh) = _system()
    graph = model.prepare(src, dst, sh, pos.shape[0], A)
    e0, f0 = energy_and_forces(model, pos, batch, cell, graph)
    model.readout_experts = ExpertReadout(model.proj_total.input_norm.normalized_shape[0], 48, 4,
                                          n_species=model.n_species).to(DEV)
    e, f = energy_and_forces(model, pos, batch, cell, graph)
    assert torch.equal(e, e0) and torch.equal(f, f0)
    assert rel_inf(e, g["energy_f64"]) < 1e-5 and rel_inf(f, g["forces_f64"]) < 1e-5
    model.readout_experts = None
    assert torch.equal(energy_and_forces(model, pos, batch, cell, graph)[1], f0)


def test_trunk_forces_training_graph_and_core():
    from fsctep_amd.capture import CapturedEnergyForces
    from fsctep_amd.core import trace_core
    from fsctep_amd.sparse import energy_and_forces
    g, model, pos, A, batch, cell, (src, dst, sh) = _system()
    _attach(model, layers=2)
    graph = model.prepare(src, dst, sh, pos.shape[0], A)
    e, f = energy_and_forces(model, pos, batch, cell, graph)
    assert rel_inf(e, g["energy_f64"]) > 1e-3                      # the experts do something
    # forces against differences of the energy along one direction
    d = torch.randn_like(pos)
    h = 1e-2
    sums = [float(energy_and_forces(model, pos + s * h * d, batch, cell, graph)[0].double().sum()) for s in (2, 1, -1, -2)]
    slope = (-sums[0] + 8 * sums[1] - 8 * sums[2] + sums[3]) / (12 * h)
    want = -float((f.double() * d.double()).sum())
    assert abs(slope - want) < 2e-2 * float(f.double().norm() * d.double().norm())
    # the force-loss step: same energies and forces, a gradient for every parameter of the experts
    model.train().requires_grad_(True)
    p = pos.clone().requires_grad_(True)
    et = model(p, A, batch, src, dst, sh, cell)
    gp, = torch.autograd.grad(et.sum(), p, create_graph=True)
    assert rel_inf(et.squeeze(-1), e) < 2e-5 and rel_inf(-gp, f) < 2e-5
    grads = torch.autograd.grad((gp ** 2).sum(), list(model.readout_experts.parameters()))
    assert all(torch.isfinite(t).all() and float(t.abs().max()) > 0 for t in grads)
    model.eval().requires_grad_(False)
    # HIP-graph replays against eager steps
    cap = CapturedEnergyForces(model, pos, batch, cell, graph)
    for k in range(4):
        q = pos + 0.01 * k
        q[k, 0] += 0.05
        ce, cf, _ = cap(q)
        ee, ef = energy_and_forces(model, q, batch, cell, graph)
        torch.cuda.synchronize()
        assert torch.equal(ce.squeeze(), ee) and torch.equal(cf, ef), k
    # the traced core at sizes other than the trace's
    core = trace_core(model, DEV)
    assert "fsctep::expert_mlp" in str(core.inlined_graph)
    p = pos.clone().requires_grad_(True)
    vec = p[dst] - p[src]
    out = core(p, A, batch, src, dst, sh, cell.reshape(1, 3, 3), vec, torch.empty(0, device=DEV))
    gp, = torch.autograd.grad(out[0].sum(), p)
    assert rel_inf(out[0].squeeze(-1), e) < 1e-6 and rel_inf(-gp, f) < 1e-5


def test_trunk_energies_in_8_bits():
    g, model, pos, A, batch, cell, (src, dst, sh) = _system()
    graph = model.prepare(src, dst, sh, pos.shape[0], A)
    with torch.no_grad():
        _attach(model, layers=2)
        full = model.readout_experts
        x = torch.randn(64, model.proj_total.input_norm.normalized_shape[0], device=DEV)
        sp = torch.arange(64, device=DEV) % model.n_species
        y, y8 = full(x, sp), full.to_8_bits()(x, sp)
        assert float((y8 - y).norm() / (y - x).norm()) < 0.05
        e = model.forward_graph(pos, batch, cell, graph)
        model.readout_experts = full.to_8_bits()
        e8 = model.forward_graph(pos, batch, cell, graph)
    assert e8.shape == e.shape and torch.isfinite(e8).all()


def test_ictd_trunk_takes_experts():
    from test_ictd_gpu import _model
    from fsctep_amd.ictd import energy_forces
    from fsctep_amd.experts import ExpertReadout
    g = load_golden("ictd_open32_c32_l2")
    model = _model(g)
    pos = torch.tensor(g["pos"], dtype=torch.float32, device=DEV)
    A = torch.tensor(g["species"], device=DEV)
    batch = torch.zeros(pos.shape[0], dtype=torch.long, device=DEV)
    cell = torch.tensor(g["cell"], dtype=torch.float32, device=DEV)
    graph = model.prepare(torch.tensor(g["edge_src"], device=DEV), torch.tensor(g["edge_dst"], device=DEV),
                          torch.tensor(g["edge_shifts"], dtype=torch.float32, device=DEV), pos.shape[0], A)
    e0, f0, _ = energy_forces(model, pos, batch, cell, graph)
    width = model.proj_total.input_norm.normalized_shape[0]
    model.readout_experts = ExpertReadout(width, 48, 4, n_species=model.n_species).to(DEV)
    e, f, _ = energy_forces(model, pos, batch, cell, graph)
    assert torch.equal(e, e0) and torch.equal(f, f0)
    _attach(model)
    e, f, _ = energy_forces(model, pos, batch, cell, graph)
    assert rel_inf(e, e0) > 1e-3 and torch.isfinite(f).all()
