"""Differentiable formulations of the light ops of the trunks, for force-loss training.

A force loss (training/trainer.py:1292-1297: F = -dE/dpos with create_graph=True, then loss.backward())
differentiates the whole energy twice, parameters included.  In ``train()`` mode the trunks therefore
build the step from:

* the conv2..n tensor products on their HIP kernels (``sparse_conv`` / ``ictd_conv``), whose C++ autograd
  gives the parameter gradients and a differentiable backward (the analogues of the reference's
  double-backward kernels, csrc/ictd_tp_cuda.cu:536-971): these carry almost all of the step's work;
* the layer norms of the energy head, with their SiLU, on the HIP op that differentiates twice, and the lookups
  by species pair on the HIP op whose gradient sums by pair (``learn_ops``);
* the functions below for the rest: edge geometry, radial basis and radial MLP, ICTD direction harmonics,
  the conv1 species-pair contraction and the readout's Gram bilinear and squared norms.  They are the same
  formulas as the inference kernels (``edge_radial.hip``, ``sparse_conv.hip`` conv1, ``ictd_conv.hip`` conv1,
  ``gram_readout.hip``, ``readout_gather.hip``) written as torch operations on the GPU, so autograd
  differentiates them to any order; the inference kernels stay the energy/force path.

Every function takes the receiver-sorted graph of ``fsctep_amd.graph`` and works on the internal layouts
(sparse x[N][13][C], ICTD x[N][M][C]).
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from .graph import Graph


def _on_ops(t) -> bool:
    """Whether a tensor is one that the HIP ops take (others, the host's and 64-bit ones, stay with torch)."""
    return t.is_cuda and t.dtype in (torch.float32, torch.bfloat16)


# ------------------------------------------------------------------ lookups (embedding.hip)
def lookup(table, index, outside: float = 0.0):
    """``table.index_select(0, index)`` of a table of any shape, its gradient summed by row in a fixed order; ``outside``
    where the ops are given an index outside the table (which index_select refuses)."""
    if not _on_ops(table) or table.numel() == 0 or table.numel() // table.shape[0] > 1 << 20:
        return table.index_select(0, index)
    from . import learn_ops
    return learn_ops.embedding(table.reshape(table.shape[0], -1), index, outside=outside).view(-1, *table.shape[1:])


# ------------------------------------------------------------------ edge geometry (edge_radial.hip)
def edge_geometry(pos, shift_vec, g: Graph):
    """vec = pos[dst] - pos[src] + shift, r = |vec|, n = vec / max(r, 1e-8) over the receiver-sorted edges
    (models/pure_cartesian_sparse_layers.py:751-756)."""
    vec = pos.index_select(0, g.dst) - pos.index_select(0, g.src) + shift_vec
    return _unit(vec)


def edge_vec_geometry(edge_vec, g: Graph):
    """The same from caller edge vectors (in the caller's edge order)."""
    return _unit(edge_vec.index_select(0, g.order.long()))


def _unit(vec):
    r = vec.norm(dim=1)
    return vec / r.clamp(min=1e-8).unsqueeze(-1), r


# ------------------------------------------------------------------ radial basis and MLP
def radial_basis(r, r_cut: float, nb: int, basis: str):
    """soft_one_hot_linspace(r, 0, r_cut, nb, basis, cutoff=True) * sqrt(nb) (e3nn's published definition,
    restated; models/pure_cartesian_sparse_layers.py:319-321).  Where a branch is cut off the value is a
    select of a finite expression, so every derivative stays finite."""
    step = r_cut / (nb + 1)
    k = torch.arange(1, nb + 1, dtype=r.dtype, device=r.device)
    x = r.unsqueeze(-1)
    if basis in ("bessel", "fourier"):
        inside = (x > 0) & (x < r_cut)
        xs = torch.where(inside, x, torch.full_like(x, 0.5 * r_cut))
        s = torch.sin(k * (math.pi / r_cut) * xs)
        if basis == "bessel":
            val = math.sqrt(2.0 / r_cut) * s / xs
        else:
            val = s / math.sqrt(0.25 + nb / 2)
        out = torch.where(inside, val, torch.zeros_like(val))
    else:
        d = (x - k * step) / step
        if basis == "gaussian":
            out = torch.exp(-d * d) / 1.12
        elif basis == "cosine":
            inside = (d > -1) & (d < 1)
            out = torch.where(inside, torch.cos(0.5 * math.pi * d), torch.zeros_like(d))
        elif basis == "smooth_finite":
            inside = (d > -1) & (d < 1)
            q = torch.where(inside, 1 - d * d, torch.ones_like(d))
            out = torch.where(inside, 1.14136 * math.exp(2.0) * torch.exp(-2.0 / q), torch.zeros_like(d))
        else:
            raise ValueError(f"radial basis {basis!r}")
    return out * math.sqrt(nb)


def radial_hidden(r, fc, r_cut: float, basis: str):
    """fc[:4](emb): silu(fc[2](silu(fc[0](emb)))) (E, 64)."""
    emb = radial_basis(r, r_cut, fc[0].in_features, basis)
    return F.silu(fc[2](F.silu(fc[0](emb))))


def radial_full(r, fc, r_cut: float, basis: str):
    """The whole radial MLP fc(emb) (E, P)."""
    return fc[4](radial_hidden(r, fc, r_cut, basis))


# ------------------------------------------------------------------ ICTD direction harmonics
_HARM = {}


def harmonics(n, lmax: int):
    """Y (E, (lmax+1)^2): block l at l^2, Y_l = sum over degree-l monomials n_x^a n_y^b n_z^c of
    multinomial * (G_l B_l) (models/ictd_irreps.py:371-402), the table edge_harmonics uses."""
    from .ictd_basis import harmonic_projection
    key = (lmax, str(n.device), n.dtype)
    if key not in _HARM:
        blocks = []
        for l in range(lmax + 1):
            exps, coef, P = harmonic_projection(l)
            M = torch.tensor(coef[:, None] * P, dtype=n.dtype, device=n.device)        # (monomials, 2l+1)
            blocks.append(([tuple(int(v) for v in e) for e in exps], M))
        _HARM[key] = blocks
    ones = torch.ones_like(n[:, 0])
    pw = []                                        # pw[axis][p] = n_axis^p, p <= lmax
    for axis in range(3):
        col = [ones]
        for _ in range(lmax):
            col.append(col[-1] * n[:, axis])
        pw.append(col)
    out = []
    for exps, M in _HARM[key]:
        mono = torch.stack([pw[0][a] * pw[1][b] * pw[2][c] for (a, b, c) in exps], dim=1)
        out.append(mono @ M)
    return torch.cat(out, dim=1)


# ------------------------------------------------------------------ conv1 (species-pair contractions)
_SPARSE_CONV1_PATHS = (0, 3, 5)       # (0,0->0), (1,0->1), (2,0->2): the paths with a rank-0 second operand


def sparse_conv1(h, n, w_last, b_last, atab, g: Graph, channels: int):
    """Sparse conv1 (models/pure_cartesian_sparse_layers.py:227-330) from the radial hidden h (E, 64):
    with W_e = h_e w_last^T + b_last in the [path][Cout][C1][C2] layout, x1 = A_src (x) n^L and x2 = A_dst,
    the message of rank L is Q_e[L][c] n^{(x)L}, Q_e[L][c] = sum_ab W_e[p_L][c][a][b] A_src[a] A_dst[b]
    = h_e . T[pair][L][c] + Tb[pair][L][c], summed to receivers / max(in-degree, 1).  The per-pair
    products run over the graph's 16-edge species-pair tiles (one batched GEMM)."""
    C, NS = channels, g.n_species
    K = h.shape[1]
    c8 = atab.shape[1]
    idx = torch.tensor(_SPARSE_CONV1_PATHS, device=h.device)
    W4 = w_last.view(6, C, c8, c8, K).index_select(0, idx)                       # (3, C, a, b, k)
    B4 = b_last.view(6, C, c8, c8).index_select(0, idx)
    T = torch.einsum("lcabk,sa,tb->stklc", W4, atab, atab).reshape(NS * NS, K, 3 * C)   # columns (L, c)
    Tb = torch.einsum("lcab,sa,tb->stlc", B4, atab, atab).reshape(NS * NS, 3 * C)
    E = h.shape[0]
    nt = g.pair_tiles.shape[0] // 17
    ids = g.pair_tiles[:16 * nt].view(nt, 16).long()
    tile_pair = g.pair_tiles[16 * nt:].long()
    valid = ids >= 0
    ht = h.index_select(0, ids.clamp(min=0).reshape(-1)).view(nt, 16, K) * valid.unsqueeze(-1).to(h.dtype)
    qt = torch.bmm(ht, lookup(T, tile_pair))                                    # (nt, 16, 3C)
    slot = torch.where(valid, ids, torch.full_like(ids, E)).reshape(-1)
    Q = h.new_zeros(E + 1, 3 * C).index_copy(0, slot, qt.reshape(-1, 3 * C))[:E]
    Q = (Q + lookup(Tb, g.edge_pair)).view(E, 3, C)
    nn_ = (n.unsqueeze(-1) * n.unsqueeze(-2)).reshape(E, 9)
    msg = torch.cat([Q[:, 0:1, :], Q[:, 1:2, :] * n.unsqueeze(-1), Q[:, 2:3, :] * nn_.unsqueeze(-1)], dim=1)
    return _receiver_mean(msg, g)


def ictd_conv1(Fe, gates, qtab, g: Graph, layout):
    """ICTD conv1 (models/pure_cartesian_ictd_layers_full.py:341-473, _o3.py:424-532): for each live path
    (l, canonical) x (0e) -> (l, canonical), whose coupling is the identity, the message of component k of
    the output block is gate[e][p] Q[pair][p] F[e][l^2 + k], Q[pair][p][o] = sum_ij W1[p][o][i][j] A_src[i]
    A_dst[j]; summed to receivers / max(in-degree, 1)."""
    E = Fe.shape[0]
    C = qtab.shape[2]
    Qe = lookup(qtab, g.edge_pair)                                                # (E, NP1, C)
    msg = Fe.new_zeros(E, layout.M, C)
    parts = []
    for i, p in enumerate(layout.conv1_paths()):
        w = gates[:, p["gate"]].unsqueeze(-1) * Qe[:, i, :]                       # (E, C)
        parts.append((p["oo"], p["d"], Fe[:, p["oy"]:p["oy"] + p["d"]].unsqueeze(-1) * w.unsqueeze(1)))
    msg = _place(msg, parts)
    return _receiver_mean(msg, g)


def _place(buf, parts):
    """buf with the (offset, width, block) parts written along dim 1 (differentiable, no in-place update
    of a tensor autograd needs)."""
    pieces, pos = [], 0
    for off, d, blk in sorted(parts, key=lambda t: t[0]):
        if off > pos:
            pieces.append(buf[:, pos:off])
        pieces.append(blk)
        pos = off + d
    if pos < buf.shape[1]:
        pieces.append(buf[:, pos:])
    return torch.cat(pieces, dim=1)


def _receiver_mean(msg, g: Graph):
    N = g.n_nodes
    deg = (g.dst_ptr[1:] - g.dst_ptr[:-1]).to(msg.dtype).clamp(min=1)
    out = msg.new_zeros((N,) + tuple(msg.shape[1:])).index_add(0, g.dst, msg)
    return out / deg.view(-1, *([1] * (msg.dim() - 1)))


# ------------------------------------------------------------------ readout (gram_readout.hip, readout_gather.hip)
def gram_bilinear(t, W, scale: float):
    """out[n][o] = scale sum_ij W[o][i][j] sum_m t[n][m][i] t[n][m][j] for t (N, D, nC), W (S, nC, nC)."""
    N, D, nC = t.shape
    S = W.shape[0]
    tw = torch.matmul(t.reshape(N * D, nC), W.permute(1, 0, 2).reshape(nC, S * nC))   # (N D, S nC): t_i W[o][i][j]
    return scale * (tw.view(N, D, S, nC) * t.unsqueeze(2)).sum(dim=(1, 3))


def readout_features(feats, Ws, scales, maps):
    """(scalars (N, S) = sum_k gram_bilinear(t_k, W_k, scale_k), sq (N, n_keys, n_layers*C)), the readout
    op's outputs: t_k are the Gram inputs the readout maps lay out (srcmap over the layers' flattened
    features), sq[n][k][l*C + c] = sum over the components m of key k of X_l[n][m][c]^2."""
    N = feats[0].shape[0]
    srcmap, _ = maps.on(feats[0].device)
    X = torch.cat([f.reshape(N, -1) for f in feats], dim=1)
    T = X.index_select(1, srcmap.long())
    nC = maps.n_layers * maps.C
    scalars, off, sqs, comp = 0, 0, [], 0
    for k, d in enumerate(maps.key_dims):
        t = T[:, off:off + d * nC].view(N, d, nC)
        scalars = scalars + gram_bilinear(t, Ws[k], scales[k])
        off += d * nC
        sqs.append(torch.cat([(f[:, comp:comp + d, :] ** 2).sum(1) for f in feats], dim=1))
        comp += d
    return scalars, torch.stack(sqs, dim=1)


# ------------------------------------------------------------------ energy head (layer_norm.hip)
def _as_made(m) -> bool:
    """Whether a call of the module is its class's forward alone: nothing hooked to it, and no forward of its own in its place."""
    return not (m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks or "forward" in vars(m))


def _plain_norm(ln) -> bool:
    """A LayerNorm over the last dimension as it was made."""
    return type(ln) is nn.LayerNorm and len(ln.normalized_shape) == 1 and _as_made(ln)


def _norm(ln, x, activation=None):
    params = [p for p in (ln.weight, ln.bias) if p is not None]
    if _on_ops(x) and x.dim() == 2 and x.shape[1] == ln.normalized_shape[0] and all(p.dtype == x.dtype for p in params):
        from . import learn_ops
        return learn_ops.layer_norm(x, ln.weight, ln.bias, ln.eps, activation)
    y = ln(x)
    return F.silu(y) if activation else y


def readout_energy(net, weighted_sum, x):
    """``weighted_sum(net(x))`` of the energy head (models/mlp.py:8-66, :117-133), differentiable twice: the layer norms and
    their SiLU on the HIP op, the products in torch.  Heads that are not as ``sparse.MainNet`` makes them run as the modules."""
    from .sparse import MainNet
    norms = [net.input_norm, *net.layer_norms] if type(net) is MainNet else []
    if (not norms or not all(_plain_norm(ln) for ln in norms) or not _as_made(net)
            or nn.modules.module._has_any_global_hook() or torch.is_autocast_enabled()):
        return weighted_sum(net(x))
    y = _norm(net.input_norm, x)
    for lin, ln in zip(net.layers, net.layer_norms):
        y = _norm(ln, lin(y), "silu")
    return weighted_sum(net.output(y))


# ------------------------------------------------------------------ expert readout (rms_norm.hip, expert_mlp.hip)
def _wide(t):
    """16-bit values in 32 bits, in which they are multiplied and summed."""
    return t.float() if t.dtype == torch.bfloat16 else t


def rms_norm(x, weight, residual=None, eps: float = 1e-6):
    """(y, z) of ``expert_ops.rms_norm``, differentiable to any order."""
    z = x if residual is None else x + residual
    v = _wide(z)
    return (v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps) * _wide(weight)).to(z.dtype), z


def _slots(index, n_experts: int):
    """Which slots have an expert, and an expert to look up for each (0 where there is none)."""
    there = (index >= 0) & (index < n_experts)
    return there, torch.where(there, index, torch.zeros_like(index)).long()


def route_weights(logits, index, score: str, renormalise: bool, scale: float):
    """The routing weights of the experts already chosen (``expert_ops.route_experts``' index), differentiable
    in the logits to any order; 0 where the index is none of the experts."""
    there, at = _slots(index, logits.shape[1])
    # a row without an expert has no weights, whatever its logits (all -inf have no softmax)
    logits = torch.where(there.any(1, keepdim=True), _wide(logits), torch.zeros((), device=logits.device))
    s = torch.softmax(logits, -1) if score == "softmax" else torch.sigmoid(logits)
    picked = torch.where(there, s.gather(1, at), torch.zeros((), device=s.device, dtype=s.dtype))
    if renormalise:
        total = picked.sum(-1, keepdim=True)
        picked = picked / torch.where(total > 0, total, torch.ones_like(total))
    return scale * picked


def expert_mlp(x, index, weight, w_in, w_out):
    """``expert_ops.expert_mlp``, differentiable to any order: every expert on every row (training
    configurations are small; the sizes follow from the tensors, so nothing waits for the GPU)."""
    E, H, f = w_out.shape
    there, at = _slots(index, E)
    share = weight.new_zeros(x.shape[0], E).scatter_add(1, at, torch.where(there, weight, torch.zeros_like(weight)))
    # what no product asks for counts for nothing, infinities and NaN included: rows without an expert, experts without a row
    zero = torch.zeros((), device=x.device, dtype=x.dtype)
    v = _wide(torch.where(there.any(1, keepdim=True), x, zero))
    chosen = torch.zeros(E, device=x.device).scatter_add(0, at.reshape(-1), there.reshape(-1).float()).view(E, 1, 1) > 0
    y = torch.zeros_like(v)
    for e, (wi, wo) in enumerate(zip(*(_wide(torch.where(chosen, w, zero)).unbind(0) for w in (w_in, w_out)))):
        a = v @ wi.t()
        y = y + share[:, e:e + 1] * ((F.silu(a[:, :f]) * a[:, f:]) @ wo.t())
    return y.to(x.dtype)
