"""Segment attention and layer norm in float64 on the CPU, one segment and one row formula at a time (numpy)."""
from __future__ import annotations

import numpy as np

__all__ = ["segment_attention_ref", "segment_attention_grads_ref", "layer_norm_ref", "layer_norm_grads_ref"]


def _segments(q_ptr, kv_ptr, nq, nk, key_mask):
    """(query rows, kept key rows) of every segment; rows outside all segments have no keys."""
    q_ptr, kv_ptr = np.clip(np.asarray(q_ptr), 0, nq), np.clip(np.asarray(kv_ptr), 0, nk)
    for b in range(len(q_ptr) - 1):
        keys = np.arange(kv_ptr[b], kv_ptr[b + 1])
        if key_mask is not None:
            keys = keys[np.asarray(key_mask)[keys].astype(bool)]
        yield np.arange(q_ptr[b], q_ptr[b + 1]), keys


def _probabilities(q, k, h, rows, keys, scale):
    s = scale * q[rows, h] @ k[keys, h * k.shape[1] // q.shape[1]].T
    top = s.max(axis=1, keepdims=True)
    e = np.exp(s - top)
    total = e.sum(axis=1, keepdims=True)
    return e / total, (top + np.log(total))[:, 0]


def segment_attention_ref(q, k, v, q_ptr, kv_ptr, key_mask=None, scale=None):
    """(out (Nq, heads, d), lse (heads, Nq)) of float64 arrays."""
    scale = q.shape[2] ** -0.5 if scale is None else scale
    out, lse = np.zeros(q.shape[:2] + (v.shape[2],)), np.full((q.shape[1], q.shape[0]), -np.inf)
    for rows, keys in _segments(q_ptr, kv_ptr, q.shape[0], k.shape[0], key_mask):
        if len(rows) and len(keys):
            for h in range(q.shape[1]):
                p, lse[h, rows] = _probabilities(q, k, h, rows, keys, scale)
                out[rows, h] = p @ v[keys, h * k.shape[1] // q.shape[1]]
    return out, lse


def segment_attention_grads_ref(go, q, k, v, q_ptr, kv_ptr, key_mask=None, scale=None):
    """(dq, dk, dv): ds = p (do v^T - sum_j p_j do v_j^T), dq = scale ds k, dk = scale ds^T q, dv = p^T do."""
    scale = q.shape[2] ** -0.5 if scale is None else scale
    dq, dk, dv = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)
    for rows, keys in _segments(q_ptr, kv_ptr, q.shape[0], k.shape[0], key_mask):
        if len(rows) and len(keys):
            for h in range(q.shape[1]):
                j = h * k.shape[1] // q.shape[1]
                p, _ = _probabilities(q, k, h, rows, keys, scale)
                dp = go[rows, h] @ v[keys, j].T
                ds = p * (dp - (p * dp).sum(axis=1, keepdims=True))
                dq[rows, h] = scale * ds @ k[keys, j]
                dk[keys, j] += scale * ds.T @ q[rows, h]
                dv[keys, j] += p.T @ go[rows, h]
    return dq, dk, dv


def layer_norm_ref(x, weight=None, bias=None, eps=1e-5, residual=None):
    """(y, s) of float64 arrays (rows, C)."""
    s = x if residual is None else x + residual
    d = s - s.mean(axis=1, keepdims=True)
    y = d / np.sqrt((d * d).mean(axis=1, keepdims=True) + eps)
    y = y if weight is None else y * weight
    return y if bias is None else y + bias, s


def layer_norm_grads_ref(gy, s, weight=None, eps=1e-5, gsum=None):
    """(gx, gweight, gbias)."""
    d = s - s.mean(axis=1, keepdims=True)
    std = np.sqrt((d * d).mean(axis=1, keepdims=True) + eps)
    xh = d / std
    t = gy if weight is None else gy * weight
    gx = (t - t.mean(axis=1, keepdims=True) - xh * (t * xh).mean(axis=1, keepdims=True)) / std
    return gx if gsum is None else gx + gsum, (gy * xh).sum(axis=0), gy.sum(axis=0)
