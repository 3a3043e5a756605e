"""Dropout from a counter-based generator, with the residual sum behind it, on the HIP library.

    y = (residual +) keep ? x * up : 0

The mask is not stored: value (row n, column f) of the last axis stays where its 16 random bits are not below
``round(65536 p)``, and is scaled by ``up = 65536 / (65536 - round(65536 p))``.  The bits come from Philox4x32 with seven
rounds (J. Salmon et al., 2011) of the counter (f // 8, n, offset) and the key seed; ``rng``, an int64 tensor (2,) on the
device, holds seed and offset and is read when the kernel runs, so a captured graph that advances ``rng[1]`` draws anew on
every replay.  The dropouts of one pass share ``rng`` and have a ``site`` each, which is added to the offset.  The backward
makes the mask again: ``rng`` has to hold then what it held in the forward (autograd refuses one that was changed in
between; advance a tensor of your own and pass a clone, as ``EGNNGlobal`` does).  What is dropped becomes 0, NaN and
infinities included.  float32 or bfloat16 (``egnn_dropout`` in include/egnn.h).  There is no reference function for this
step, and no CPU path: ROCm tensors only.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _capi
from ._capi import EgnnDropout, check
from .fused import _dtype_code, _ptr, _recorded, _stream
from .layer_norm import MAX_WIDTH, _rows

__all__ = ["Dropout", "dropout", "dropout_forward", "dropout_backward", "DropoutFn"]


class Dropout(NamedTuple):
    """A dropout's probability, seed and offset, and number among those that share them: what
    :func:`pymolecular_amd.layer_norm.layer_norm_dropout` takes."""
    p: float
    rng: torch.Tensor
    site: int = 0


def check_drop(drop: Dropout, dev) -> EgnnDropout:
    """The C struct, of arguments that have been looked at."""
    p, rng, site = drop
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"the probability of a dropout must be 0 to 1 (got {p})")
    if rng.dtype != torch.int64 or tuple(rng.shape) != (2,) or not rng.is_contiguous() or rng.device != dev:
        raise ValueError(f"rng must hold seed and offset, (2,) int64 on {dev} (got {tuple(rng.shape)} {rng.dtype} on "
                         f"{rng.device})")
    return EgnnDropout(rng.data_ptr(), site, p)


def dropout_forward(x, p, rng, residual=None, site=0):
    """``egnn_dropout``: dropout of ``x``, or ``residual`` + dropout of ``x`` in the dtype of their sum."""
    r = _capi.ext().dropout(x, p, rng, site, residual)
    if r is not None:
        return r
    # a tensor needs a conversion, or an argument is refused
    if not x.is_cuda:
        raise RuntimeError("x must be a ROCm device tensor: the dropout has no CPU path")
    _dtype_code(x.dtype)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"x needs a last axis of 1 to {MAX_WIDTH} values (got {tuple(x.shape)})")
    if residual is not None and (residual.shape != x.shape or residual.device != x.device):
        raise ValueError(f"residual must have x's shape {tuple(x.shape)} and device (got {tuple(residual.shape)})")
    drop = check_drop(Dropout(p, rng, site), x.device)
    if residual is not None and residual.dtype != x.dtype:
        dt = torch.promote_types(x.dtype, residual.dtype)
        _dtype_code(dt)
        x, residual = x.to(dt), residual.to(dt)
    x2, r2 = _rows(x), None if residual is None else _rows(residual)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    with torch.cuda.device(x.device):   # (its stream may not be of the current one)
        check("egnn_dropout",
              _capi.lib().egnn_dropout(drop, _dtype_code(x.dtype), x2.shape[0], x2.shape[1], x2.data_ptr(), x2.stride(0),
                                       _ptr(r2), 0 if r2 is None else r2.stride(0), y.data_ptr(), _stream(x.device)))
    return y


def dropout_backward(gy, p, rng, site=0):
    """The gradient of ``x`` (that of the residual is ``gy``): the forward's mask on the gradient of ``y``."""
    return dropout_forward(gy, p, rng, site=site)


class DropoutFn(torch.autograd.Function):
    """``y = DropoutFn.apply(x, p, rng, residual, site)``; saves ``rng`` alone."""

    @staticmethod
    def forward(ctx, x, p, rng, residual, site):
        y = dropout_forward(x, p, rng, residual, site)
        ctx.save_for_backward(rng)
        ctx.p, ctx.site, ctx.xdt, ctx.rdt = p, site, x.dtype, None if residual is None else residual.dtype
        return y

    @staticmethod
    def backward(ctx, gy):
        rng, = ctx.saved_tensors
        gx = None
        if ctx.needs_input_grad[0]:
            gx = dropout(gy, ctx.p, rng, site=ctx.site)   # (linear in gy: it can be differentiated again)
            gx = gx if gx.dtype == ctx.xdt else gx.to(ctx.xdt)
        gr = None
        if ctx.rdt is not None and ctx.needs_input_grad[3]:
            gr = gy if gy.dtype == ctx.rdt else gy.to(ctx.rdt)
        return gx, None, None, gr, None


def dropout(x: torch.Tensor, p: float, rng: torch.Tensor, residual: Optional[torch.Tensor] = None,
            site: int = 0) -> torch.Tensor:
    """Dropout of ``x``, or ``residual`` + dropout of ``x`` (module docstring).  Differentiable in ``x`` and the
    residual."""
    if not (torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad))):
        r = _capi.ext().dropout(x, p, rng, site, residual)
        if r is not None:   # (neither a tensor that needs a conversion, nor a call that has to be recorded)
            return r
        if not _recorded(x, residual):
            return dropout_forward(x, p, rng, residual, site)
    return DropoutFn.apply(x, p, rng, residual, site)
