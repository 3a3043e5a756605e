"""Rows of a table by token, times a scale, and the table's gradient, on the HIP library.

    out_i = scale * weight[tokens_i],    grad_weight[v] = scale * sum of grad_out_i over the i with tokens_i = v

Tokens (int32 or int64, any shape) name node types, elements, residues or fragments.  The gradient sorts them first, so that
each row of ``grad_out`` is read once and each row of the table is written once, with sums in a fixed order (float32; the
parts of a long run in 64 bits).  A token outside the table has a row of zeros and no gradient; the row ``padding`` is read
as any other and gets no gradient.  Rows are float32 or bfloat16; a float32 table beside bfloat16 rows keeps the gradients in
float32 (``egnn_embed_fwd`` / ``egnn_embed_bwd`` in include/egnn.h).  There is no reference function for this step, and no CPU
path: ROCm tensors only.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _capi
from ._capi import EgnnEmbedDims, check
from .fused import _dtype_code, _first_order, _ptr, _recorded, _stream
from .layer_norm import MAX_WIDTH, _rows

__all__ = ["embedding", "embedding_forward", "embedding_backward", "EmbeddingFn"]


def _check(tokens, vocab, width, scale, padding):
    if not tokens.is_cuda:
        raise RuntimeError("tokens must be a ROCm device tensor: the embedding has no CPU path")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"tokens must be int32 or int64 (got {tokens.dtype})")
    if not 1 <= width <= MAX_WIDTH or not 1 <= vocab < 1 << 31 or vocab * width >= 1 << 40:
        raise ValueError(f"the table must have 1 to 2^31 - 1 rows of 1 to {MAX_WIDTH} values, below 2^40 in all (got "
                         f"{vocab}, {width})")
    if tokens.numel() >= 1 << 31:
        raise ValueError(f"{tokens.numel()} tokens: at most 2^31 - 1")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite (got {scale})")
    if padding is not None and not 0 <= padding < vocab:
        raise ValueError(f"padding must be a row of the table, 0 to {vocab - 1} (got {padding})")


def _dims(tokens, vocab, width, dt, table_dt, scale) -> EgnnEmbedDims:
    return EgnnEmbedDims(tokens.numel(), vocab, width, _dtype_code(dt), table_dt != dt, tokens.dtype == torch.int64, scale)


def embedding_forward(tokens, weight, scale=1.0, dtype=None):
    """``egnn_embed_fwd``: (\\*tokens.shape, width) rows of ``dtype`` (None: the weight's)."""
    dtype = weight.dtype if dtype is None else dtype
    r = _capi.ext().embed_forward(tokens, weight, scale, dtype)
    if r is not None:
        return r
    # a tensor needs a conversion, or an argument is refused
    if weight.dim() != 2:
        raise ValueError(f"weight must be (vocab, width) (got {tuple(weight.shape)})")
    _check(tokens, *weight.shape, scale, None)
    if weight.device != tokens.device:
        raise ValueError(f"weight is on {weight.device}, tokens on {tokens.device}")
    _dtype_code(dtype)
    w = weight if weight.dtype in (dtype, torch.float32) else weight.to(torch.float32)
    if w.dtype != dtype and dtype == torch.float32:
        w = w.to(dtype)
    w = _rows(w)
    t = tokens.contiguous()
    out = torch.empty((*tokens.shape, weight.shape[1]), dtype=dtype, device=tokens.device)
    with torch.cuda.device(t.device):   # (its stream may not be of the current one)
        check("egnn_embed_fwd",
              _capi.lib().egnn_embed_fwd(_dims(t, *weight.shape, dtype, w.dtype, scale), t.data_ptr(), w.data_ptr(), w.stride(0),
                                         out.data_ptr(), _stream(t.device)))
    return out


def embedding_backward(grad_out, tokens, vocab, scale=1.0, padding=None, dtype=None):
    """``egnn_embed_bwd``: the gradient (vocab, width) of the table in ``dtype`` (None: that of ``grad_out``)."""
    dtype = grad_out.dtype if dtype is None else dtype
    r = _capi.ext().embed_backward(grad_out, tokens, vocab, scale, -1 if padding is None else padding, dtype)
    if r is not None:
        return r
    if grad_out.dim() != tokens.dim() + 1 or grad_out.shape[:-1] != tokens.shape or grad_out.device != tokens.device:
        raise ValueError(f"grad_out must be tokens' shape {tuple(tokens.shape)} and the width, on its device (got "
                         f"{tuple(grad_out.shape)})")
    _check(tokens, vocab, grad_out.shape[-1], scale, padding)
    dt = grad_out.dtype
    _dtype_code(dt)
    table_dt = dt if dtype == dt else torch.float32
    g, t = _rows(grad_out), tokens.contiguous()
    d = _dims(t, vocab, grad_out.shape[-1], dt, table_dt, scale)
    gw = torch.empty((vocab, grad_out.shape[-1]), dtype=table_dt, device=t.device)
    L = _capi.lib()
    nbytes = L.egnn_embed_bwd_workspace_bytes(d)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=t.device) if nbytes else None
    with torch.cuda.device(t.device):   # (its stream may not be of the current one)
        check("egnn_embed_bwd",
              L.egnn_embed_bwd(d, -1 if padding is None else padding, g.data_ptr(), g.stride(0), t.data_ptr(), gw.data_ptr(),
                               _ptr(ws), nbytes, _stream(t.device)))
    return gw if gw.dtype == dtype else gw.to(dtype)


class EmbeddingFn(torch.autograd.Function):
    """``out = EmbeddingFn.apply(tokens, weight, scale, padding, dtype)``; saves the tokens alone."""

    @staticmethod
    def forward(ctx, tokens, weight, scale, padding, dtype):
        out = embedding_forward(tokens, weight, scale, dtype)
        ctx.save_for_backward(tokens)
        ctx.vocab, ctx.scale, ctx.padding, ctx.dtype = weight.shape[0], scale, padding, weight.dtype
        return out

    @staticmethod
    def backward(ctx, gout):
        tokens, = ctx.saved_tensors
        grad = embedding_backward(gout, tokens, ctx.vocab, ctx.scale, ctx.padding, ctx.dtype)
        return None, *_first_order((grad,), gout), None, None, None


def embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding: Optional[int] = None,
              dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``scale`` times the rows of ``weight`` (vocab, width) that ``tokens`` name (module docstring), in ``dtype`` (None:
    the weight's).  Differentiable in the weight."""
    if padding is not None and not 0 <= padding < weight.shape[0]:
        raise ValueError(f"padding must be a row of the table, 0 to {weight.shape[0] - 1} (got {padding})")
    if not (torch.is_grad_enabled() and weight.requires_grad):
        r = _capi.ext().embed_forward(tokens, weight, scale, weight.dtype if dtype is None else dtype)
        if r is not None:   # (neither a tensor that needs a conversion, nor a call that has to be recorded)
            return r
        if not _recorded(weight):
            return embedding_forward(tokens, weight, scale, dtype)
    return EmbeddingFn.apply(tokens, weight, scale, padding, dtype)
