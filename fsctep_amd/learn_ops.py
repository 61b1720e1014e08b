"""Operators of the training step: ``torch.ops.fsctep.layer_norm`` and ``embedding``, differentiable as a loss on
forces needs them.

The ops are registered in C++ by ``libfsctep_torch.so`` (``csrc/torch_learn_ops.cpp``) over the C ABI of
``libfsctep_hip.so``: device, Meta and autograd kernels, launches on the current stream, no host synchronisation, no
CPU implementation.  ``fsctep_amd.train_ops`` builds the trunks' training step with them (the reference's LayerNorm
and SiLU, models/mlp.py:8-66, and its lookups by species, models/pure_cartesian_sparse_layers.py:258-259);
``fsctep_amd.optim`` has the optimiser.

    layer_norm(x, weight=None, bias=None, eps=1e-5, activation=None) -> y
    embedding(table, index, scale=1.0, outside=0.0) -> rows

``layer_norm`` differentiates twice (rows, weight, bias), ``embedding`` to any order (table); a third derivative of
``layer_norm`` and forward-mode derivatives raise.
"""

from __future__ import annotations

from . import _lib

_lib.load_torch_ops()

import torch  # noqa: E402

ACTIVATIONS = {None: 0, "silu": 1}


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, activation: str | None = None):
    """``act((x - mean) / sqrt(var + eps) * weight + bias)`` of (rows, width) rows, float32 or bfloat16, any row
    stride; ``weight`` and ``bias`` float32 or of the rows' type (None: 1 and 0); ``activation``: None or "silu"."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation {activation!r}: expected None or 'silu'")
    return torch.ops.fsctep.layer_norm(x, weight, bias, float(eps), ACTIVATIONS[activation], False)[0]


def embedding(table, index, scale: float = 1.0, outside: float = 0.0):
    """``scale * table[index]``, (\\*index.shape, width), of a (rows, width) table, float32 or bfloat16, for an index of
    any shape, int32 or int64; ``outside``, without a gradient, where the index lies outside the table (-1: padding).  The
    table's gradient sums the rows of each token in 32 bits and in a fixed order."""
    if index.dim() == 1:
        return torch.ops.fsctep.embedding(table, index, float(scale), float(outside))
    rows = torch.ops.fsctep.embedding(table, index.reshape(-1), float(scale), float(outside))
    return rows.view(*index.shape, rows.shape[1])
