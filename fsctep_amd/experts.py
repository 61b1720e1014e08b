"""Mixture of experts on the per-atom invariants, between a trunk's readout features and its energy head.

    model.readout_experts = ExpertReadout(model.proj_total.input_norm.normalized_shape[0], hidden=640, n_experts=8,
                                          n_species=model.n_species)

adds to the invariants x (N, width), layer by layer, ``x + sum_j weight_j expert_j(norm(x))`` with the experts
chosen per atom by a router (``expert_ops``): from a table of scores by atomic number (``n_species`` rows), or,
without ``n_species``, from the normalised rows themselves.  A choice by atomic number does not change as atoms
move, so energies stay smooth functions of the positions and forces conserve them; a choice by rows steps where an
atom changes experts, which is for energies and for training on them, not for dynamics.  The layers' outputs start
at zero, so a trained trunk keeps its energies when one is attached.  The reference has no counterpart; trunks
without one run as before.

* energies and forces: the fused operators, whose gradient with respect to the rows gives the forces;
* training the experts on energies: the same with the parameters' gradients (a trunk in ``eval()`` mode, whose own
  parameters have none there);
* training on forces (the trunks' ``train()`` step): ``differentiable=True``, the twice differentiable torch form
  on the experts that the fused router chose;
* energies alone of many candidates (screening, Monte Carlo): ``ExpertReadout.to_8_bits()``, rows and weights in 8
  bits, no gradient;
* the layers in bfloat16: ``ExpertReadout.bfloat16()``, on float32 rows too (what a layer adds is bfloat16, the rows
  themselves stay as they are).
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import expert_ops as X

ROW_TYPES = (torch.float32, torch.bfloat16)


class _OwnTypes(nn.Module):
    """Buffers that keep their types where a program casts the parameters (``.bfloat16()`` and the like)."""

    def _apply(self, fn, recurse=True):
        before = dict(self._buffers)
        super()._apply(fn, recurse)
        for name, b in before.items():
            if self._buffers[name].dtype != b.dtype:
                self._buffers[name] = b.to(self._buffers[name].device)
        return self


class ExpertLayer(_OwnTypes):
    """Parameters of one layer: norm weight (width,), gate (n_experts, width) or, by atomic number, (n_species,
    n_experts), w_in (n_experts, 2 hidden, width), w_out (n_experts, width, hidden, zero at first) and the balance
    bias (n_experts,), a float32 buffer that moves which experts are chosen and not what they weigh."""

    def __init__(self, width: int, hidden: int, n_experts: int, n_species: int | None = None):
        super().__init__()
        self.norm = nn.Parameter(torch.ones(width))
        self.gate = nn.Parameter(torch.randn(n_experts, width) / math.sqrt(width) if n_species is None
                                 else torch.randn(n_species, n_experts))
        self.w_in = nn.Parameter(torch.randn(n_experts, 2 * hidden, width) / math.sqrt(width))
        self.w_out = nn.Parameter(torch.zeros(n_experts, width, hidden))
        self.register_buffer("balance", torch.zeros(n_experts))

    @torch.no_grad()
    def rebalance(self, index, rate: float = 0.001):
        """One step of the balance rule: experts chosen less often than the mean gain ``rate``, the others lose
        it (``index``: the router's choices of a batch)."""
        n = self.balance.shape[0]
        flat = index.reshape(-1).long()
        count = self.balance.new_zeros(n + 1).index_add_(0, torch.where((flat < 0) | (flat > n), n, flat),
                                                         torch.ones_like(flat, dtype=self.balance.dtype))[:n]
        self.balance += rate * torch.sign(count.mean() - count)


class Router:
    """How an expert readout chooses: the settings of ``expert_ops.route_experts`` and where the logits come from."""

    def __init__(self, n_experts, k, score, groups, groups_kept, group_best, renormalise, scale, n_species):
        if not 1 <= k <= n_experts:
            raise ValueError("expert readout: k must be 1 to n_experts")
        if score not in X.SCORES:
            raise ValueError(f"score {score!r}: expected one of {sorted(X.SCORES)}")
        self.k, self.score, self.n_species = int(k), score, None if n_species is None else int(n_species)
        self.groups, self.groups_kept, self.group_best = int(groups), int(groups_kept), int(group_best)
        self.renormalise, self.scale = bool(renormalise), float(scale)

    def rows_of(self, species, below):
        """Rows of the layers' tables for the atoms and which atoms have none (None: all have one).  ``below``: what the
        caller's atomic numbers are known to lie under; where that is not within the tables they are looked at."""
        if self.n_species is None:
            return None, None
        if species is None:
            raise ValueError("this expert readout chooses by atomic number: pass species (N,)")
        if below is not None and below <= self.n_species:
            return species, None
        none = (species < 0) | (species >= self.n_species)
        return species.masked_fill(none, 0), none.unsqueeze(1)

    def logits(self, layer, y, species, none=None):
        """Of an atom without a row NaN, which the router passes on to what the atom becomes."""
        if self.n_species is None:
            return F.linear(y, layer.gate)
        l = layer.gate.index_select(0, species)
        return l if none is None else l.masked_fill(none, math.nan)

    def choose(self, layer, logits):
        return X.route_experts(logits, self.k, score=self.score, bias=layer.balance, groups=self.groups,
                               groups_kept=self.groups_kept, group_best=self.group_best,
                               renormalise=self.renormalise, scale=self.scale)


class ExpertReadout(nn.Module):
    """``layers`` expert layers on rows (N, width); ``k`` of ``n_experts`` experts a row, scores ``softmax`` or
    ``sigmoid``, optional groups (``groups``, ``groups_kept``, ``group_best``), weights renormalised and scaled as
    ``expert_ops.route_experts`` does; ``n_species``: choice by atomic number.  Parameters in float32 or, after
    ``.bfloat16()``, in bfloat16; rows in either."""

    def __init__(self, width: int, hidden: int, n_experts: int, k: int = 2, layers: int = 1, score: str = "softmax",
                 groups: int = 1, groups_kept: int = 1, group_best: int = 1, renormalise: bool = True,
                 scale: float = 1.0, eps: float = 1e-6, n_species: int | None = None):
        super().__init__()
        if min(width, hidden, n_experts, layers) < 1:
            raise ValueError("ExpertReadout: width, hidden, n_experts and layers must be at least 1")
        self.router = Router(n_experts, k, score, groups, groups_kept, group_best, renormalise, scale, n_species)
        self.eps = float(eps)
        self.layers = nn.ModuleList([ExpertLayer(width, hidden, n_experts, n_species) for _ in range(layers)])

    def forward(self, x, species=None, differentiable: bool = False, species_below: int | None = None):
        """(N, width) -> (N, width); ``species``: atomic numbers (N,), below n_species (an atom with another becomes NaN).
        ``differentiable``: twice differentiable (force losses).  ``species_below``: what the caller knows ``species`` to
        lie under from 0 on, so that they need not be looked at."""
        if x.dtype not in ROW_TYPES:
            raise ValueError(f"expert readout: rows are float32 or bfloat16, got {x.dtype}")
        rows = self.router.rows_of(species, species_below)
        if differentiable:
            return self._forward_train(x, rows)
        own = self.layers[0].norm.dtype
        if x.dtype != own:
            out = x
            for layer in self.layers:
                y, _ = X.rms_norm(out.to(own), layer.norm, eps=self.eps)
                index, weight = self.router.choose(layer, self.router.logits(layer, y, *rows))
                out = out + X.expert_mlp(y, index, weight, layer.w_in, layer.w_out)
            return out.to(x.dtype)
        z, add = x, None
        for layer in self.layers:
            y, z = X.rms_norm(x, layer.norm, eps=self.eps) if add is None else X.rms_norm(add, layer.norm, z, self.eps)
            index, weight = self.router.choose(layer, self.router.logits(layer, y, *rows))
            add = X.expert_mlp(y, index, weight, layer.w_in, layer.w_out)
        return z + add

    def _forward_train(self, x, rows):
        from . import train_ops as T
        own, given = self.layers[0].norm.dtype, x.dtype
        for layer in self.layers:
            y, _ = T.rms_norm(x.to(own), layer.norm, eps=self.eps)
            logits = self.router.logits(layer, y, *rows)
            with torch.no_grad():
                index, _ = self.router.choose(layer, logits.detach())
            weight = T.route_weights(logits, index, self.router.score, self.router.renormalise,
                                     self.router.scale)
            x = x + T.expert_mlp(y, index, weight, layer.w_in, layer.w_out)
        return x.to(given)

    def to_8_bits(self) -> "ExpertReadoutQ8":
        return ExpertReadoutQ8(self)


class ExpertReadoutQ8(nn.Module):
    """An ``ExpertReadout``'s weights in 8 bits, made once: energies without gradients.  The rows between the
    layers are held in bfloat16; the router sees the values that the 8-bit rows stand for."""

    def __init__(self, full: ExpertReadout):
        super().__init__()
        self.router, self.eps = full.router, full.eps
        self.layers = nn.ModuleList()
        for layer in full.layers:
            m = _OwnTypes()
            m.register_buffer("norm", layer.norm.detach().float().clone())
            m.register_buffer("gate", layer.gate.detach().float().clone())
            m.register_buffer("balance", layer.balance.detach().clone())
            for name in ("w_in", "w_out"):
                codes, scale = X.to_codes(getattr(layer, name))
                m.register_buffer(name, codes)
                m.register_buffer(name + "_scale", scale)
            self.layers.append(m)

    @torch.no_grad()
    def forward(self, x, species=None, differentiable: bool = False, species_below: int | None = None):
        if differentiable:
            raise RuntimeError("the 8-bit expert readout has no gradient; train the ExpertReadout it was made from")
        rows = self.router.rows_of(species, species_below)
        z, add = x.to(torch.bfloat16), None
        for m in self.layers:
            q, scale, z = X.rms_norm_q8(z, m.norm, None, self.eps) if add is None else \
                X.rms_norm_q8(add, m.norm, z, self.eps)
            index, weight = self.router.choose(m, self.router.logits(m, q * scale.unsqueeze(-1), *rows))
            add = X.expert_mlp_q8(q, scale, index, weight, m.w_in, m.w_in_scale, m.w_out, m.w_out_scale)
        return (z.float() + add.float()).to(x.dtype)
