"""Norm of every head of queries and keys, and their rotation by position, in one pass on the HIP library.

    y = x / sqrt(mean x^2 + eps) * weight,    (a, b) -> (a cos - b sin, b cos + a sin)  for the pairs of y's first values

``q`` is (N, heads, d), ``k`` (N, kv_heads, d), with a weight (d,) each (None: 1).  The first ``rotary_dim`` values of a head
(None: all of them) are turned by ``positions[n] * base ** (-2 i / rotary_dim)``, i the pair's number, so that the product of
a query and a key depends on how far apart they are: residues of a chain.  Pairs are the first half and the second half of
those values, or neighbours if ``interleaved``.  Positions are int32 or int64 and may be far (|position| <= 2^32 to 2^-29
turns, further ones in proportion); without positions nothing is turned.  float32 or bfloat16 with fp32 sums, even head widths
up to 128, parts of one projection's rows (``qkv[:, :heads]``) read where they lie.  The backward recomputes what it needs from
the inputs (``egnn_qk_fwd`` / ``egnn_qk_bwd`` in include/egnn.h); a head whose gradient is 0 throughout takes no part in it and
may hold anything.  :func:`qk_norm_rotary_attention` puts :func:`pymolecular_amd.segment_attention.segment_attention` behind it,
where masked keys and rows outside every segment are such heads.  There is no reference function for this step, and no CPU path:
ROCm tensors only.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _capi
from ._capi import EgnnQkDims, EgnnQkStrides, check
from .fused import _as, _dtype_code, _first_order, _ptr, _recorded, _stream
from .layer_norm import _param_dtype
from .segment_attention import _parts, segment_attention_backward, segment_attention_forward

__all__ = ["qk_norm_rotary", "qk_norm_rotary_forward", "qk_norm_rotary_backward", "QKNormRotaryFn",
           "qk_norm_rotary_attention", "QKNormRotaryAttentionFn"]

MAX_HEAD_DIM, MAX_HEADS = 128, 4096


def _check(q, k, q_weight, k_weight, positions, base, rotary_dim, eps):
    if not q.is_cuda:
        raise RuntimeError("q must be a ROCm device tensor: the norm and rotation of heads have no CPU path")
    _dtype_code(q.dtype)
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"q and k must be (N, heads, d) and (N, kv_heads, d) (got {tuple(q.shape)}, {tuple(k.shape)})")
    d = q.shape[2]
    if d % 2 or not 2 <= d <= MAX_HEAD_DIM:
        raise ValueError(f"the head width must be even, 2 to {MAX_HEAD_DIM} (got {d})")
    if not 1 <= q.shape[1] <= MAX_HEADS or not 1 <= k.shape[1] <= MAX_HEADS or q.shape[0] >= 1 << 31:
        raise ValueError(f"1 to {MAX_HEADS} heads and fewer than 2^31 rows (got {tuple(q.shape)}, {tuple(k.shape)})")
    if k.dtype != q.dtype or k.device != q.device:
        raise TypeError(f"q and k must have one dtype and device (got {q.dtype}, {k.dtype} on {q.device}, {k.device})")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (tuple(w.shape) != (d,) or w.device != q.device):
            raise ValueError(f"{name} must be ({d},) on {q.device} (got {tuple(w.shape)} on {w.device})")
    if rotary_dim % 2 or not 0 <= rotary_dim <= d:
        raise ValueError(f"rotary_dim must be even, 0 to {d} (got {rotary_dim})")
    if positions is None:
        if rotary_dim:
            raise ValueError("a rotation needs positions")
    elif positions.dtype not in (torch.int32, torch.int64) or tuple(positions.shape) != (q.shape[0],) or positions.device != q.device:
        raise ValueError(f"positions must be ({q.shape[0]},) of int32 or int64 on {q.device} (got {tuple(positions.shape)} "
                         f"{positions.dtype})")
    if not 1 <= base < math.inf or not 0 <= eps < math.inf:
        raise ValueError(f"base must be 1 or more, eps 0 or more, both finite (got {base}, {eps})")


def _rotary(q, positions, rotary_dim) -> int:
    if rotary_dim is None:
        return 0 if positions is None else q.shape[-1]
    return rotary_dim


def _call(q, k, q_weight, k_weight, positions, base, rotary_dim, interleaved, eps):
    """(q, k, q_weight, k_weight, positions) as the library takes them, and its dims."""
    _check(q, k, q_weight, k_weight, positions, base, rotary_dim, eps)
    pdt = _param_dtype(q.dtype, *(None if w is None else w.dtype for w in (q_weight, k_weight)))
    q, k = (t if t.stride(2) == 1 else t.contiguous() for t in (q, k))
    positions = positions if positions is None else positions.contiguous()
    d = EgnnQkDims(q.shape[0], q.shape[1], k.shape[1], q.shape[2], rotary_dim, interleaved, _dtype_code(q.dtype),
                   pdt != q.dtype, positions is not None and positions.dtype == torch.int64, eps, base)
    return q, k, _as(q_weight, pdt), _as(k_weight, pdt), positions, d


def qk_norm_rotary_forward(q, k, q_weight=None, k_weight=None, positions=None, base=10000.0, rotary_dim=None,
                           interleaved=False, eps=1e-6):
    """``egnn_qk_fwd``: returns ``(q', k')``."""
    rotary_dim = _rotary(q, positions, rotary_dim)
    r = _capi.ext().qk_forward(q, k, q_weight, k_weight, positions, base, rotary_dim, interleaved, eps)
    if r is not None:
        return r
    # a tensor needs a conversion, or an argument is refused
    q, k, qw, kw, pos, d = _call(q, k, q_weight, k_weight, positions, base, rotary_dim, interleaved, eps)
    out = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k)]
    s = EgnnQkStrides(*(x for t in (q, k, *out) for x in t.stride()[:2]))
    with torch.cuda.device(q.device):   # (its stream may not be of the current one)
        check("egnn_qk_fwd", _capi.lib().egnn_qk_fwd(d, s, q.data_ptr(), k.data_ptr(), _ptr(qw), _ptr(kw), _ptr(pos),
                                                     out[0].data_ptr(), out[1].data_ptr(), _stream(q.device)))
    return tuple(out)


def qk_norm_rotary_backward(gq_out, gk_out, q, k, q_weight=None, k_weight=None, positions=None, base=10000.0,
                            rotary_dim=None, interleaved=False, eps=1e-6, into=None):
    """``egnn_qk_bwd``: returns ``(gq, gk, gq_weight, gk_weight)``, the last two None without weights.  ``into``: two
    tensors to write the first two to (parts of one buffer, say), of the inputs' shapes and dtype, rows and heads apart."""
    rotary_dim = _rotary(q, positions, rotary_dim)
    wdt = [None if w is None else w.dtype for w in (q_weight, k_weight)]
    r = _capi.ext().qk_backward(gq_out, gk_out, q, k, q_weight, k_weight, positions, base, rotary_dim, interleaved, eps,
                                None if into is None else list(into))
    if r is not None:
        return r
    q, k, qw, kw, pos, d = _call(q, k, q_weight, k_weight, positions, base, rotary_dim, interleaved, eps)
    for name, g, t in (("gq_out", gq_out, q), ("gk_out", gk_out, k)):
        if g.shape != t.shape or g.device != t.device:
            raise ValueError(f"{name} must have the shape {tuple(t.shape)} and device of its input (got {tuple(g.shape)})")
    gq_out, gk_out = (g if g.dtype == q.dtype else g.to(q.dtype) for g in (gq_out, gk_out))
    gq_out, gk_out = (g if g.stride(2) == 1 else g.contiguous() for g in (gq_out, gk_out))
    if into is None:
        grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k)]
    else:
        grads = list(into)
        for g, t in zip(grads, (q, k)):
            if (g.shape != t.shape or g.dtype != t.dtype or g.device != t.device or g.stride(2) != 1
                    or g.stride(1) < t.shape[2] or g.stride(0) < t.shape[1] * t.shape[2]):
                raise ValueError("into must hold tensors of the inputs' shapes and dtype, rows and heads apart")
    pdt = torch.float32 if d.f32_params else q.dtype
    gw = [None if w is None else torch.empty((q.shape[2],), dtype=pdt, device=q.device) for w in (qw, kw)]
    L = _capi.lib()
    nbytes = L.egnn_qk_bwd_workspace_bytes(d) if qw is not None or kw is not None else 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    out = [g.stride()[:2] for g in (gq_out, gk_out, *grads)]
    s = EgnnQkStrides(*q.stride()[:2], *k.stride()[:2], 0, 0, 0, 0, *(x for t in out for x in t))
    with torch.cuda.device(q.device):   # (its stream may not be of the current one)
        check("egnn_qk_bwd",
              L.egnn_qk_bwd(d, s, gq_out.data_ptr(), gk_out.data_ptr(), q.data_ptr(), k.data_ptr(), _ptr(qw), _ptr(kw),
                            _ptr(pos), grads[0].data_ptr(), grads[1].data_ptr(), _ptr(gw[0]), _ptr(gw[1]), _ptr(ws), nbytes,
                            _stream(q.device)))
    return (*grads, *(_as(g, t) for g, t in zip(gw, wdt)))


class QKNormRotaryFn(torch.autograd.Function):
    """``q', k' = QKNormRotaryFn.apply(q, k, q_weight, k_weight, positions, base, rotary_dim, interleaved, eps)``; saves
    its inputs."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, *how):
        ctx.save_for_backward(q, k, q_weight, k_weight, positions)
        ctx.how = how
        return qk_norm_rotary_forward(q, k, q_weight, k_weight, positions, *how)

    @staticmethod
    def backward(ctx, gq, gk):
        q, k, qw, kw, positions = ctx.saved_tensors
        grads = qk_norm_rotary_backward(gq, gk, q, k, qw, kw, positions, *ctx.how)
        return (*_first_order(grads, gq, gk, q, k, qw, kw), None, None, None, None, None)


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                   k_weight: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                   base: float = 10000.0, rotary_dim: Optional[int] = None, interleaved: bool = False,
                   eps: float = 1e-6):
    """``(q', k')``: heads normed and turned (module docstring).  Differentiable in q, k and the weights."""
    tensors = (q, k, q_weight, k_weight)
    how = (base, _rotary(q, positions, rotary_dim), interleaved, eps)
    if not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)):
        r = _capi.ext().qk_forward(*tensors, positions, *how)
        if r is not None:   # (neither a tensor that needs a conversion, nor a call that has to be recorded)
            return r
        if not _recorded(*tensors):
            return qk_norm_rotary_forward(*tensors, positions, *how)
    return QKNormRotaryFn.apply(*tensors, positions, *how)


class QKNormRotaryAttentionFn(torch.autograd.Function):
    """``out = QKNormRotaryAttentionFn.apply(qkv, heads, seg_ptr, key_mask, scale, q_weight, k_weight, positions, base,
    rotary_dim, interleaved, eps)``: all gradients of the projection's rows are written into one buffer."""

    @staticmethod
    def forward(ctx, qkv, heads, seg_ptr, key_mask, scale, q_weight, k_weight, positions, *how):
        q, k, v = _parts(qkv, heads)
        q, k = qk_norm_rotary_forward(q, k, q_weight, k_weight, positions, *how)
        out, lse = segment_attention_forward(q, k, v, seg_ptr, None, key_mask, scale)
        ctx.save_for_backward(qkv, q, k, out, lse, seg_ptr, key_mask, q_weight, k_weight, positions)
        ctx.heads, ctx.scale, ctx.how = heads, scale, how
        return out

    @staticmethod
    def backward(ctx, gout):
        qkv, q, k, out, lse, seg_ptr, key_mask, qw, kw, positions = ctx.saved_tensors
        grad = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        (q0, k0, v), (gq0, gk0, gv) = _parts(qkv, ctx.heads), _parts(grad, ctx.heads)
        if qkv.shape[2] % 8:   # widths that the attention pads
            gq, gk, g = segment_attention_backward(gout, q, k, v, out, lse, seg_ptr, None, key_mask, ctx.scale)
            gv.copy_(g)
        else:
            gq, gk = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
            segment_attention_backward(gout, q, k, v, out, lse, seg_ptr, None, key_mask, ctx.scale, into=(gq, gk, gv))
        *_, gqw, gkw = qk_norm_rotary_backward(gq, gk, q0, k0, qw, kw, positions, *ctx.how, into=(gq0, gk0))
        grad, gqw, gkw = _first_order((grad, gqw, gkw), gout, qkv, qw, kw)
        return grad, None, None, None, None, gqw, gkw, None, None, None, None, None


def qk_norm_rotary_attention(qkv: torch.Tensor, heads: int, seg_ptr: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                             k_weight: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                             key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                             base: float = 10000.0, rotary_dim: Optional[int] = None, interleaved: bool = False,
                             eps: float = 1e-6) -> torch.Tensor:
    """:func:`pymolecular_amd.segment_attention.segment_attention_qkv` of a projection (N, heads + 2 kv_heads, d) whose
    queries and keys are normed and turned first (module docstring): (N, heads, d).  Differentiable in ``qkv`` and the
    weights."""
    tensors = (qkv, q_weight, k_weight)
    how = (base, rotary_dim, interleaved, eps)
    if (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)) or _recorded(*tensors):
        return QKNormRotaryAttentionFn.apply(qkv, heads, seg_ptr, key_mask, scale, q_weight, k_weight, positions, *how)
    q, k, v = _parts(qkv, heads)
    q, k = qk_norm_rotary_forward(q, k, q_weight, k_weight, positions, *how)
    return segment_attention_forward(q, k, v, seg_ptr, None, key_mask, scale, need_lse=False)[0]
