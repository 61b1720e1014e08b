"""Operators of the expert readout: ``torch.ops.fsctep.rms_norm`` / ``route_experts`` / ``expert_mlp`` and their
8-bit forms.

The ops are registered in C++ by ``libfsctep_torch.so`` (``csrc/torch_expert_ops.cpp``) over the C ABI of
``libfsctep_hip.so``: device, Meta and autograd kernels, launches on the current stream, no host
synchronisation, no CPU implementation.  The reference has no counterpart (its energy head is one MainNet,
models/mlp.py:8-66).

    rms_norm(x, weight, residual=None, eps=1e-6) -> (y, z)
    rms_norm_q8(x, weight, residual=None, eps=1e-6) -> (codes, scale, z)
    route_experts(logits, k, score="softmax", bias=None, groups=1, groups_kept=1, group_best=1,
                  renormalise=True, scale=1.0) -> (index, weight)
    expert_mlp(x, index, weight, w_in, w_out) -> y
    expert_mlp_q8(codes, scale, index, weight, w_in, w_in_scale, w_out, w_out_scale) -> y (bfloat16)
    to_codes(w) -> (codes, scale)

``rms_norm``, ``route_experts`` and ``expert_mlp`` have gradients (rows, residual, norm weight; logits; rows,
routing weights, experts' weights); a gradient of a gradient raises, ``train_ops.expert_readout`` is the twice
differentiable form of the whole.  The 8-bit forms have no gradient: they serve energies.
"""

from __future__ import annotations

from . import _lib

_lib.load_torch_ops()

import torch  # noqa: E402

SCORES = {"softmax": 0, "sigmoid": 1}


def rms_norm(x, weight, residual=None, eps: float = 1e-6):
    """``z = x + residual`` (``x`` itself without a residual), ``y = z / sqrt(mean z^2 + eps) * weight`` of
    (rows, width) rows, float32 or bfloat16, any row stride; ``weight`` float32 or of the rows' type.  Returns
    (y, z): the next layer's residual is z."""
    y, z, _ = torch.ops.fsctep.rms_norm(x, weight, residual, float(eps))
    return y, (x if residual is None else z)


def rms_norm_q8(x, weight, residual=None, eps: float = 1e-6):
    """``rms_norm`` with y in 8 bits: (codes int8, scale float32 (rows,), z), y = codes * scale."""
    q, scale, z = torch.ops.fsctep.rms_norm_q8(x, weight, residual, float(eps))
    return q, scale, (x if residual is None else z)


def route_experts(logits, k: int, score: str = "softmax", bias=None, groups: int = 1, groups_kept: int = 1,
                  group_best: int = 1, renormalise: bool = True, scale: float = 1.0):
    """The k experts of each row with the largest ``s + bias`` (s the softmax or sigmoid of the logits; ties to
    the lowest expert) and their weights ``scale * s / sum of the chosen s`` (``/ 1`` without ``renormalise``):
    (index int32 (rows, k), weight float32 (rows, k)).  With ``groups`` only the experts of the ``groups_kept``
    groups whose ``group_best`` largest biased scores have the largest sum are open.  A logit of -inf bars an
    expert; slots left over have index -1 and weight 0."""
    if score not in SCORES:
        raise ValueError(f"score {score!r}: expected one of {sorted(SCORES)}")
    return torch.ops.fsctep.route_experts(logits, bias, int(k), SCORES[score], int(groups), int(groups_kept),
                                          int(group_best), bool(renormalise), float(scale))


def expert_mlp(x, index, weight, w_in, w_out):
    """``y_t = sum_j weight_tj w_out[e] (silu(w_in[e][:F] x_t) * (w_in[e][F:] x_t))`` with e = index_tj, for rows
    x (T, H), index (int32) and weight (float32) (T, k), w_in (E, 2F, H) and w_out (E, H, F) of x's type (float32
    or bfloat16).  An index outside [0, E) adds nothing.

    Sums are held in 32 bits.  float32 products are made of 16-bit parts: 24 bits of every operand, or, where an expert has
    more than about 80 rows, 22 bits of values down to 2^-17 of the largest of their row (of the rows) or output column (of
    the weights).  In bfloat16 the hidden values and their gradients are rounded to bfloat16 between the products where an
    expert has more than about 32 rows, which makes the error about 1.4 times that of the one rounding at the end; with
    fewer rows they stay in float32."""
    return torch.ops.fsctep.expert_mlp(x, index, weight, w_in, w_out)


def expert_mlp_q8(codes, scale, index, weight, w_in, w_in_scale, w_out, w_out_scale):
    """``expert_mlp`` on 8-bit rows (``rms_norm_q8``) and 8-bit weights (``to_codes``), bfloat16 out; the hidden
    values are held in 8 bits with a unit for each row and 128 columns."""
    return torch.ops.fsctep.expert_mlp_q8(codes, scale, index, weight, w_in, w_in_scale, w_out, w_out_scale)


def to_codes(w):
    """8-bit codes of weights with a scale for each row of the last dimension: (int8, float32), w = codes * scale
    to half a code."""
    w = w.detach().float()
    scale = w.abs().amax(-1) / 127
    # (a scale next to the smallest number is a rounded one: its codes may come out above 127)
    return torch.round(w / torch.where(scale > 0, scale, 1.0).unsqueeze(-1)).clamp(-127, 127).to(torch.int8), scale
