"""Expert readout in plain 64-bit torch on the CPU, written from the formulas: the oracle of rms_norm, route_experts,
expert_mlp and their 8-bit forms."""

from __future__ import annotations

import math

import torch


def rms_norm(x, weight, residual=None, eps=1e-6, held=None):
    """(y, z); ``held``: the type that z is rounded to before it is normalised (None: not rounded)."""
    x, weight = x.double(), weight.double()
    z = x if residual is None else x + residual.double()
    if held is not None:
        z = z + (z.detach().to(held).double() - z.detach())
    return z / torch.sqrt((z ** 2).mean(1, keepdim=True) + eps) * weight, z


def codes(y):
    """(codes, scale) of rows y: scale = max |y| / 127, code the nearest whole number of y / scale."""
    top = y.abs().amax(-1, keepdim=True)
    unit = torch.where(top > 0, top / 127, torch.ones_like(top))
    return torch.round(y / unit), (top / 127).squeeze(-1)


def scores(logits, score):
    logits = logits.double()
    if score == "sigmoid":
        return torch.sigmoid(logits)
    m = logits.max(1, keepdim=True).values
    e = torch.exp(logits - torch.where(m == -math.inf, torch.zeros_like(m), m))
    t = e.sum(1, keepdim=True)
    return e / torch.where(t > 0, t, torch.ones_like(t))


def choose(c, k, groups=1, kept=1, best=1):
    """Row by row: the k experts of largest c, ties to the lowest, -1 where none is left; c -inf: barred."""
    out = []
    for row in c.tolist():
        n, per = len(row), len(row) // groups
        if groups > 1:
            rank = []
            for g in range(groups):
                top = sorted((v for v in row[g * per:(g + 1) * per] if v > -math.inf), reverse=True)[:best]
                rank.append(sum(top) if top else -math.inf)
            keep = sorted(range(groups), key=lambda g: (-rank[g], g))[:kept]
            row = [v if i // per in keep else -math.inf for i, v in enumerate(row)]
        order = [i for i in sorted(range(n), key=lambda i: (-row[i], i)) if row[i] > -math.inf][:k]
        out.append(order + [-1] * (k - len(order)))
    return torch.tensor(out, dtype=torch.int32).reshape(len(out), k)


def weights(logits, index, score, renormalise=True, scale=1.0):
    s = scores(logits, score)
    there = index >= 0
    picked = s.gather(1, index.clamp(min=0).long()) * there
    if renormalise:
        t = picked.sum(1, keepdim=True)
        picked = picked / torch.where(t > 0, t, torch.ones_like(t))
    return scale * picked


def route_gradient(logits, index, score, renormalise, scale, u):
    """dL/dlogits by the formula, u = dL/dweights: with n the weights over ``scale``, renormalised weights have
    ds_j s_j = scale n_j (u_j - sum u n), others scale n_j u_j; then sigmoid: (ds_j s_j)(1 - s_j), softmax:
    ds_i s_i - s_i sum_j ds_j s_j."""
    s = scores(logits, score)
    n = weights(logits, index, score, renormalise)
    d = scale * n * (u - (u * n).sum(1, keepdim=True) if renormalise else u)
    at = index.clamp(min=0).long()
    if score == "sigmoid":
        return torch.zeros_like(s).scatter_add_(1, at, d * (1 - s.gather(1, at)) * (index >= 0))
    dl = torch.zeros_like(s).scatter_add_(1, at, d * (index >= 0))
    return dl if renormalise else dl - s * d.sum(1, keepdim=True)     # renormalised: the sum is zero


def expert_mlp(x, index, weight, w_in, w_out, group=None):
    """Slot by slot; ``group``: hidden columns that share an 8-bit unit (None: not rounded)."""
    x, weight, w_in, w_out = (t.double() for t in (x, weight, w_in, w_out))
    f = w_out.shape[2]
    y = torch.zeros_like(x)
    for e in range(w_out.shape[0]):
        row, slot = torch.nonzero(index == e, as_tuple=True)
        a = x[row] @ w_in[e].T
        gate, up = a[:, :f], a[:, f:]
        h = gate * torch.sigmoid(gate) * up
        if group is not None:
            parts = []
            for lo in range(0, f, group):
                q, s = codes(h[:, lo:lo + group])
                parts.append(q * s.unsqueeze(1))
            h = torch.cat(parts, 1)
        y = y.index_add(0, row, (h @ w_out[e].T) * weight[row, slot].unsqueeze(1))
    return y
