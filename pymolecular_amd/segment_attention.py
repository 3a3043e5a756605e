"""Attention over all nodes of each graph of a batch, forward and backward, on the HIP library.

The graphs lie back to back (segment offsets, as in :mod:`pymolecular_amd.graph_build`): no padding, no mask between
graphs.  ``q`` is (Nq, heads, d), ``k`` and ``v`` are (Nk, kv_heads, d) with ``heads`` a multiple of ``kv_heads`` (head
``h`` uses key head ``h * kv_heads // heads``); queries ``q_ptr[b]:q_ptr[b + 1]`` attend the keys
``kv_ptr[b]:kv_ptr[b + 1]``, by default the same nodes:

    s_ij = scale q_i . k_j,    out_i = sum_j softmax_j(s_ij) v_j      over the keys j of i's graph with key_mask[j]

A query without any key left gets 0 and takes part in no gradient.  float32 or bfloat16, any head width up to 128;
parts of one projection's rows (``qkv[:, :heads]``) are read where they lie.  There is no reference function for this
step, and no CPU path: ROCm tensors only (``egnn_attn_fwd`` / ``egnn_attn_bwd`` in include/egnn.h).
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _capi
from ._capi import EgnnAttnDims, EgnnAttnStrides, check
from .fused import _dtype_code, _first_order, _ptr, _recorded, _stream

__all__ = ["segment_attention", "segment_attention_qkv", "segment_attention_forward", "segment_attention_backward",
           "SegmentAttentionFn", "SegmentAttentionQKVFn"]

MAX_HEAD_DIM = 128


def _heads(t: torch.Tensor, group: int = 1) -> torch.Tensor:
    """``t`` (n, heads, d) if the kernels can read it where it lies, else a contiguous copy: unit-stride heads, 16-byte
    aligned, rows apart (or all the same one) by at most 16 MiB, the ``group`` heads on one key head by 512 MiB.  A width
    that is not a multiple of 8 is padded with zeros (which change neither the scores nor the output's own columns)."""
    d, e = t.shape[2], t.element_size()
    if d % 8:
        return torch.nn.functional.pad(t, (0, 8 - d % 8))
    rs, hs = t.stride(0), t.stride(1)
    if (t.stride(2) == 1 and rs * e % 16 == 0 and hs * e % 16 == 0 and t.data_ptr() % 16 == 0
            and (rs == 0 or d <= rs <= (1 << 24) // e) and (group - 1) * hs * e <= 1 << 29):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _check(q, k, v, q_ptr, kv_ptr, key_mask, scale):
    if not q.is_cuda:
        raise RuntimeError("q must be a ROCm device tensor: the segment attention has no CPU path")
    _dtype_code(q.dtype)
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or q.shape[2] != k.shape[2]:
        raise ValueError("q, k, v must be (Nq, heads, d), (Nk, kv_heads, d), (Nk, kv_heads, d): got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if not 1 <= q.shape[2] <= MAX_HEAD_DIM:
        raise ValueError(f"the head width must be 1 to {MAX_HEAD_DIM} (got {q.shape[2]})")
    if k.shape[1] < 1 or q.shape[1] < 1 or q.shape[1] % k.shape[1]:
        raise ValueError(f"{q.shape[1]} query heads are not a multiple of {k.shape[1]} key heads")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q, k and v must have one dtype (got {q.dtype}, {k.dtype}, {v.dtype})")
    for name, p in (("q_ptr", q_ptr), ("kv_ptr", kv_ptr)):
        if p.dtype != torch.int32 or p.dim() != 1 or p.numel() < 1 or not p.is_contiguous():
            raise ValueError(f"{name} must hold n_seg + 1 contiguous int32 offsets")
    if q.shape[1] >= 1 << 31 or q_ptr.numel() > 1 << 31:   # what the library counts in 32 bits
        raise ValueError(f"{q.shape[1]} heads, {q_ptr.numel()} offsets: at most 2^31 - 1 heads and segments")
    if q_ptr.numel() != kv_ptr.numel():
        raise ValueError(f"q_ptr and kv_ptr have {q_ptr.numel()} and {kv_ptr.numel()} offsets")
    if kv_ptr is q_ptr and q.shape[0] != k.shape[0]:
        raise ValueError(f"{q.shape[0]} queries and {k.shape[0]} keys need a kv_ptr")
    if key_mask is not None and (key_mask.dtype not in (torch.bool, torch.uint8) or tuple(key_mask.shape) != (k.shape[0],)):
        raise ValueError(f"key_mask must be ({k.shape[0]},) of bool or uint8")
    for name, t in (("k", k), ("v", v), ("q_ptr", q_ptr), ("kv_ptr", kv_ptr), ("key_mask", key_mask)):
        if t is not None and t.device != q.device:
            raise ValueError(f"{name} is on {t.device}, q on {q.device}")
    if not math.isfinite(scale) or scale == 0:
        raise ValueError(f"scale must be finite and not 0 (got {scale})")


def _scale(q, scale) -> float:
    return float(q.shape[-1]) ** -0.5 if scale is None and q.dim() and q.shape[-1] else float(scale or 0.0)


def _defaults(q, q_ptr, kv_ptr, key_mask, scale):
    if key_mask is not None and not key_mask.is_contiguous():
        key_mask = key_mask.contiguous()
    return q_ptr if kv_ptr is None else kv_ptr, key_mask, _scale(q, scale)


def _dims(q, k, q_ptr, scale) -> EgnnAttnDims:
    return EgnnAttnDims(q.shape[0], k.shape[0], q_ptr.numel() - 1, q.shape[1], k.shape[1], q.shape[2],
                        _dtype_code(q.dtype), scale)


def _workspace(nbytes, dev):
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def segment_attention_forward(q, k, v, q_ptr, kv_ptr=None, key_mask=None, scale=None, need_lse=True):
    """``egnn_attn_fwd``: returns ``(out, lse)``; ``lse`` (heads, Nq) float32 is what
    :func:`segment_attention_backward` needs (None where ``need_lse`` is false)."""
    r = _capi.ext().attn_forward(q, k, v, q_ptr, kv_ptr, key_mask, _scale(q, scale), need_lse)
    if r is not None:
        return r
    # a tensor needs a conversion, or an argument is refused
    kv_ptr, key_mask, scale = _defaults(q, q_ptr, kv_ptr, key_mask, scale)
    _check(q, k, v, q_ptr, kv_ptr, key_mask, scale)
    d = q.shape[2]
    group = q.shape[1] // k.shape[1]
    q, k, v = _heads(q, group), _heads(k), _heads(v)
    dims = _dims(q, k, q_ptr, scale)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=q.device) if need_lse else None
    L = _capi.lib()
    nbytes = L.egnn_attn_fwd_workspace_bytes(dims)
    ws = _workspace(nbytes, q.device)
    s = EgnnAttnStrides(q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1), out.stride(0),
                        out.stride(1))
    check("egnn_attn_fwd", L.egnn_attn_fwd(dims, s, q.data_ptr(), k.data_ptr(), v.data_ptr(), q_ptr.data_ptr(),
                                           kv_ptr.data_ptr(), _ptr(key_mask), out.data_ptr(), _ptr(lse), _ptr(ws),
                                           nbytes, _stream(q.device)))
    return (out if q.shape[2] == d else out[:, :, :d]), lse


def segment_attention_backward(gout, q, k, v, out, lse, q_ptr, kv_ptr=None, key_mask=None, scale=None, into=None):
    """``egnn_attn_bwd``: returns ``(grad_q, grad_k, grad_v)`` from the forward's ``out`` and ``lse``.  ``into``: three
    tensors to write them to (parts of one buffer, say), of the inputs' shapes and dtype with 16-byte aligned
    unit-stride heads."""
    r = _capi.ext().attn_backward(gout, q, k, v, out, lse, q_ptr, kv_ptr, key_mask, _scale(q, scale),
                                  None if into is None else list(into))
    if r is not None:
        return r
    kv_ptr, key_mask, scale = _defaults(q, q_ptr, kv_ptr, key_mask, scale)
    _check(q, k, v, q_ptr, kv_ptr, key_mask, scale)
    if gout.shape != q.shape or out.shape != q.shape:
        raise ValueError(f"gout and out must have q's shape {tuple(q.shape)} (got {tuple(gout.shape)}, {tuple(out.shape)})")
    if lse.dtype != torch.float32 or tuple(lse.shape) != (q.shape[1], q.shape[0]) or not lse.is_contiguous():
        raise ValueError(f"lse must be the forward's ({q.shape[1]}, {q.shape[0]}) float32 statistics")
    if any(t.device != q.device for t in (gout, out, lse)):
        raise ValueError("gout, out and lse must be on q's device")
    d = q.shape[2]
    group = q.shape[1] // k.shape[1]
    gout = _heads(gout if gout.dtype == q.dtype else gout.to(q.dtype), group)
    out = _heads(out if out.dtype == q.dtype else out.to(q.dtype), group)
    q, k, v = _heads(q, group), _heads(k), _heads(v)
    dims = _dims(q, k, q_ptr, scale)
    if into is None:
        grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v)]
    else:
        grads = list(into)
        for g, t in zip(grads, (q, k, v)):
            if g.shape != t.shape or g.dtype != t.dtype or g.device != t.device or _heads(g) is not g or g.stride(0) < g.shape[2]:
                raise ValueError("into must hold tensors of the inputs' shapes and dtype with 16-byte aligned heads")
    L = _capi.lib()
    nbytes = L.egnn_attn_bwd_workspace_bytes(dims)
    ws = _workspace(nbytes, q.device)
    s = EgnnAttnStrides(*(x for t in (q, k, v, out, gout, *grads) for x in (t.stride(0), t.stride(1))))
    check("egnn_attn_bwd", L.egnn_attn_bwd(dims, s, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                           lse.data_ptr(), gout.data_ptr(), q_ptr.data_ptr(), kv_ptr.data_ptr(),
                                           _ptr(key_mask), *(g.data_ptr() for g in grads), _ptr(ws), nbytes,
                                           _stream(q.device)))
    return tuple(g if g.shape[2] == d else g[:, :, :d] for g in grads)


class SegmentAttentionFn(torch.autograd.Function):
    """``out = SegmentAttentionFn.apply(q, k, v, q_ptr, kv_ptr, key_mask, scale)``; saves its inputs, the output and
    one statistic a row and head, and recomputes the probabilities in the backward."""

    @staticmethod
    def forward(ctx, q, k, v, q_ptr, kv_ptr, key_mask, scale):
        out, lse = segment_attention_forward(q, k, v, q_ptr, kv_ptr, key_mask, scale)
        ctx.save_for_backward(q, k, v, out, lse, q_ptr, kv_ptr, key_mask)
        ctx.scale = scale
        return out

    @staticmethod
    def backward(ctx, gout):
        q, k, v, out, lse, q_ptr, kv_ptr, key_mask = ctx.saved_tensors
        grads = segment_attention_backward(gout, q, k, v, out, lse, q_ptr, kv_ptr, key_mask, ctx.scale)
        return (*_first_order(grads, gout, q, k, v), None, None, None, None)


class SegmentAttentionQKVFn(torch.autograd.Function):
    """``out = SegmentAttentionQKVFn.apply(qkv, heads, seg_ptr, key_mask, scale)``: queries, keys and values in the rows
    of one projection; the three gradients are written into the rows of one buffer, the projection's gradient."""

    @staticmethod
    def forward(ctx, qkv, heads, seg_ptr, key_mask, scale):
        out, lse = segment_attention_forward(*_parts(qkv, heads), seg_ptr, None, key_mask, scale)
        ctx.save_for_backward(qkv, out, lse, seg_ptr, key_mask)
        ctx.heads, ctx.scale = heads, scale
        return out

    @staticmethod
    def backward(ctx, gout):
        qkv, out, lse, seg_ptr, key_mask = ctx.saved_tensors
        parts = _parts(qkv, ctx.heads)
        if qkv.shape[2] % 8:   # widths that are padded
            grad = torch.cat(segment_attention_backward(gout, *parts, out, lse, seg_ptr, None, key_mask, ctx.scale), dim=1)
        else:
            grad = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
            segment_attention_backward(gout, *parts, out, lse, seg_ptr, None, key_mask, ctx.scale,
                                       into=_parts(grad, ctx.heads))
        return (*_first_order((grad,), gout, qkv), None, None, None, None)


def _parts(qkv, heads):
    """(q, k, v) in the rows of one projection (N, heads + 2 kv_heads, d)."""
    if qkv.dim() != 3 or not 0 < heads < qkv.shape[1] or (qkv.shape[1] - heads) % 2:
        raise ValueError(f"qkv must be (N, heads + 2 kv_heads, d) with {heads} heads: got {tuple(qkv.shape)}")
    kv = (qkv.shape[1] - heads) // 2
    return qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]


def _inference(q, k, v, q_ptr, kv_ptr, key_mask, scale):
    """The output alone, or None where the call has to be recorded (the native entry refuses such tensors by itself)."""
    r = _capi.ext().attn_forward(q, k, v, q_ptr, kv_ptr, key_mask, _scale(q, scale), False)
    if r is not None:
        return r[0]
    if _recorded(q, k, v):
        return None
    return segment_attention_forward(q, k, v, q_ptr, kv_ptr, key_mask, scale, need_lse=False)[0]


def segment_attention_qkv(qkv: torch.Tensor, heads: int, seg_ptr: torch.Tensor, key_mask: Optional[torch.Tensor] = None,
                          scale: Optional[float] = None) -> torch.Tensor:
    """:func:`segment_attention` of each segment over itself, with queries, keys and values in the rows of one projection:
    ``qkv`` (N, heads + 2 kv_heads, d) -> (N, heads, d)."""
    if not (torch.is_grad_enabled() and qkv.requires_grad):
        r = _inference(*_parts(qkv, heads), seg_ptr, None, key_mask, scale)
        if r is not None:
            return r
    return SegmentAttentionQKVFn.apply(qkv, heads, seg_ptr, key_mask, scale)


def segment_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_ptr: torch.Tensor,
                      kv_ptr: Optional[torch.Tensor] = None, key_mask: Optional[torch.Tensor] = None,
                      scale: Optional[float] = None) -> torch.Tensor:
    """Attention of each segment's queries over its keys (module docstring), (Nq, heads, d); ``scale`` defaults to
    d ** -0.5.  Differentiable in q, k and v."""
    if not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)):
        r = _inference(q, k, v, q_ptr, kv_ptr, key_mask, scale)
        if r is not None:
            return r
    return SegmentAttentionFn.apply(q, k, v, q_ptr, kv_ptr, key_mask, scale)
