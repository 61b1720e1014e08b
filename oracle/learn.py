"""The training step's operators in 64 bits (layer norm, lookup, AdamW), and the sizes that bound their roundings.

Test infrastructure only.  ``norm_sizes`` gives, for every output of the layer norm and its two backward passes, the
sum of the magnitudes of the terms it is made of: a sum of n terms in 32 bits is off by at most about n 2^-24 times
that."""

from __future__ import annotations

import numpy as np
import torch


def layer_norm(x, w, b, eps, silu):
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    u = c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    if w is not None:
        u = u * w
    if b is not None:
        u = u + b
    return u * torch.sigmoid(u) if silu else u


def norm_all(x, w, b, eps, silu, dy, v, vw=None, vb=None):
    """{output: value} of y, dx, dw, db and of the backward of (dx, dw, db) with cotangents (v, vw, vb)."""
    x, dy = x.detach().double().requires_grad_(True), dy.detach().double().requires_grad_(True)
    w, b = (None if t is None else t.detach().double().requires_grad_(True) for t in (w, b))
    y = layer_norm(x, w, b, eps, silu)
    out = {"y": y}
    ins = {"x": x} | ({} if w is None else {"w": w}) | ({} if b is None else {"b": b})
    first = dict(zip(ins, torch.autograd.grad(y, list(ins.values()), dy, create_graph=True)))
    out |= {"d" + k: g for k, g in first.items()}
    ends = [(first["x"], v)] + [(first[k], c) for k, c in (("w", vw), ("b", vb)) if c is not None]
    ins["dy"] = dy
    second = torch.autograd.grad([e for e, _ in ends], list(ins.values()), [c.double() for _, c in ends], allow_unused=True)
    out |= {"g" + k: torch.zeros_like(t) if g is None else g for (k, t), g in zip(ins.items(), second)}
    return {k: t.detach() for k, t in out.items()}


def norm_sizes(x, w, b, eps, silu, dy, v, vw=None, vb=None):
    """{output: sum of the magnitudes of its terms}, laid out as ``norm_all``."""
    x, dy, v = x.detach().double(), dy.detach().double().abs(), v.detach().double().abs()
    one, zero = torch.ones(x.shape[1], dtype=torch.float64, device=x.device), torch.zeros(x.shape[1], dtype=torch.float64, device=x.device)
    w, b = one if w is None else w.detach().double().abs(), zero if b is None else b.detach().double().abs()
    vw, vb = (zero if t is None else t.detach().double().abs() for t in (vw, vb))

    def mean(t):
        return t.mean(-1, keepdim=True)

    c = x - mean(x)
    r = 1 / torch.sqrt(mean(c * c) + eps)
    zh = (c * r).abs()
    u = zh * w + b
    # SiLU's derivatives are at most 1.1 and 0.5; the sigmoid passes on the argument's relative error, u times as large
    d1, d2, more = (1.1, 0.5, 1 + u) if silu else (1.0, 0.0, 1.0)
    du = dy * d1 * more
    g = du * w
    q = r * (v + mean(v) + zh * mean(v * zh))
    a = w * q + vw * zh + vb
    e = dy * d2 * a * more
    k = e * w + du * vw + r * (g * mean(v * zh) + v * mean(g * zh))
    turn = mean(g * v) + mean(g) * mean(v) + mean(g * zh) * mean(v * zh)
    return {"y": u * more, "dx": r * (g + mean(g) + zh * mean(g * zh)), "dw": (du * zh).sum(0), "db": du.sum(0),
            "gx": r * (k + mean(k) + zh * mean(k * zh)) + r * r * zh * turn, "gw": (du * q + e * zh).sum(0),
            "gb": e.sum(0), "gdy": d1 * a * more}


def embedding(table, index, scale):
    index = index.long()
    there = (index >= 0) & (index < table.shape[0])
    if table.shape[0] == 0:
        return table.new_zeros(*index.shape, table.shape[1])
    return torch.where(there.unsqueeze(-1), scale * table[torch.where(there, index, 0)], 0.0)


def embedding_grad(dy, index, rows, scale):
    index = index.long()
    there = (index >= 0) & (index < rows)
    out = torch.zeros(rows, dy.shape[1], dtype=torch.float64, device=dy.device)
    return out.index_add_(0, index[there], dy[there].double()) * scale


def adamw(p, g, m, v, step, lr, betas, eps, weight_decay, clip=1.0):
    """(p, m, v) after one step from 64-bit values; ``step``: steps taken before."""
    b1, b2 = betas
    t = step + 1
    g = g * clip
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return p * (1 - lr * weight_decay) - lr / (1 - b1 ** t) * m / (np.sqrt(v) / np.sqrt(1 - b2 ** t) + eps), m, v


# ------------------------------------------------------------------ 8-bit states
# The grid of a code: the numbers (1 + f / 2^F) 2^e, F fraction bits, the largest code at 1 (f 0, e 0), code 0 at 0.
def grid(root: bool):
    fraction, top = (4, 255) if root else (3, 127)
    steps = np.arange(top + 1) - top
    e = steps >> fraction
    g = (1 + (steps - (e << fraction)) / 2.0 ** fraction) * 2.0 ** e
    g[0] = 0.0
    return g


def hash32(place, step):
    h = (place.astype(np.uint64) * 0x9E3779B1 + np.uint64(step) * np.uint64(0x6A09E667)) & np.uint64(0xFFFFFFFF)
    h ^= h >> np.uint64(16)
    h = (h * np.uint64(0xBB67AE85)) & np.uint64(0xFFFFFFFF)
    h ^= h >> np.uint64(15)
    h = (h * np.uint64(0x3C6EF373)) & np.uint64(0xFFFFFFFF)
    return h ^ (h >> np.uint64(16))


def encode(x, step, root: bool):
    """(codes, scales) of float32 values, every operation in float32: where between its two neighbours on the grid a
    value lies, compared with a random number."""
    n = x.shape[0]
    codes, scales = np.zeros(n, np.uint8), np.zeros(-(-n // 256), np.float32)
    g = grid(root)
    bits = 19 if root else 20
    for k in range(scales.shape[0]):
        part = x[256 * k:256 * k + 256]
        top = np.abs(part).max()
        if top < np.float32(2.0) ** -100:
            codes[256 * k:256 * k + 256] = 0 if root else np.where(part < 0, 128, 0)
            continue
        scales[k] = top
        y = np.minimum(np.abs(part) * (np.float32(1) / top), np.float32(1)).astype(np.float64)
        h = hash32(np.arange(256 * k, 256 * k + part.shape[0]), step)
        add = ((h >> np.uint64(13)) if root else (h & np.uint64(0xFFFFF))).astype(np.float64) / 2.0 ** bits
        # below the first code the grid goes on in the same way; what would be rounded to a code below 1 is 0
        low = np.searchsorted(g[1:], y, side="right")          # number of codes >= 1 at or below y
        below = np.where(low > 0, g[low], 0)
        above = g[np.minimum(low + 1, len(g) - 1)]
        share = np.where(low > 0, (y - below) / np.where(above > below, above - below, 1), 0)
        up = share + add >= 1
        # between code 0's place on the continued grid and code 1
        fraction = 4 if root else 3
        step1 = 2.0 ** np.floor(np.log2(g[1])) / 2 ** fraction
        zero_place = g[1] - step1 if np.log2(g[1]) % 1 else g[1] - step1 / 2
        under = (low == 0) & (y >= zero_place) & ((y - zero_place) / (g[1] - zero_place) + add >= 1)
        c = low + (up & (low > 0)) + under
        c = np.minimum(c, len(g) - 1)
        if root:
            c = np.where(y > 0, np.maximum(c, 1), 0)
        else:
            c = c + np.where(part < 0, 128, 0)
        codes[256 * k:256 * k + 256] = c
    return codes, scales


def decode(codes, scales, root: bool):
    g = grid(root).astype(np.float32)
    size = codes if root else codes & 127
    y = g[size]
    if not root:
        y = np.where(codes >= 128, -y, y)
    return (y * np.repeat(scales, 256)[:codes.shape[0]]).astype(np.float32)
