"""Table rows by token and the table's gradient in float64 on the CPU (numpy)."""
from __future__ import annotations

import numpy as np

__all__ = ["embedding_ref", "embedding_grad_ref"]


def embedding_ref(tokens, weight, scale=1.0):
    """tokens (n,), weight (vocab, C): (n, C); zeros for tokens outside the table."""
    tokens = np.asarray(tokens, dtype=np.int64)
    inside = (tokens >= 0) & (tokens < weight.shape[0])
    return np.where(inside[:, None], scale * weight[np.where(inside, tokens, 0)], 0.0)


def embedding_grad_ref(grad_out, tokens, vocab, scale=1.0, padding=None):
    """(vocab, C)."""
    tokens = np.asarray(tokens, dtype=np.int64)
    inside = (tokens >= 0) & (tokens < vocab)
    gw = np.zeros((vocab, grad_out.shape[1]))
    if inside.any():
        order = np.flatnonzero(inside)
        order = order[np.argsort(tokens[order], kind="stable")]
        names, first = np.unique(tokens[order], return_index=True)
        gw[names] = np.add.reduceat(grad_out[order], first, axis=0)
    if padding is not None:
        gw[padding] = 0.0
    return scale * gw
