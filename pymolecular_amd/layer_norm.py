"""Layer norm over the last axis, with the residual sum in front of it, on the HIP library.

    s = x (+ residual),   y = (s - mean s) / sqrt(var s + eps) * weight + bias

``y`` is made from the unrounded sum; with a residual the sum is returned too (what the next residual adds to).  The
backward takes the gradients of both and makes the weight's and the bias's over all rows in a fixed order
(``egnn_norm_fwd`` / ``egnn_norm_bwd`` in include/egnn.h).  float32 or bfloat16 with fp32 statistics, any width up to 2^20 and
any row stride.  ``y`` and the sum have the dtype of ``x + residual``; weight and bias enter, and their gradients leave, in
float32 where they have another dtype than the rows (float32 parameters beside bfloat16 activations).  With a dropout in
front of the sum (:func:`layer_norm_dropout`, ``egnn_norm_drop_fwd`` / ``_bwd``), ``s = residual + dropout(x)``, the mask
is that of :mod:`pymolecular_amd.dropout`.  There is no reference function for this step, and no CPU path: ROCm tensors
only.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _capi
from ._capi import EgnnNormDims, check
from .fused import _as, _dtype_code, _first_order, _ptr, _recorded, _stream

__all__ = ["layer_norm", "layer_norm_forward", "layer_norm_backward", "LayerNormFn", "layer_norm_dropout",
           "layer_norm_dropout_forward", "layer_norm_dropout_backward", "LayerNormDropoutFn"]

MAX_WIDTH = 1 << 20


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as (rows, C) with unit-stride rows; a copy only where it has to be."""
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _check(x, weight, bias, residual, eps):
    if not x.is_cuda:
        raise RuntimeError("x must be a ROCm device tensor: the layer norm has no CPU path")
    _dtype_code(x.dtype)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"x needs a last axis of 1 to {MAX_WIDTH} values (got {tuple(x.shape)})")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and (tuple(p.shape) != (x.shape[-1],) or p.device != x.device):
            raise ValueError(f"{name} must be ({x.shape[-1]},) on {x.device} (got {tuple(p.shape)} on {p.device})")
    if residual is not None and (residual.shape != x.shape or residual.device != x.device):
        raise ValueError(f"residual must have x's shape {tuple(x.shape)} and device (got {tuple(residual.shape)})")
    if not 0 <= eps < float("inf"):
        raise ValueError(f"eps must be finite and not negative (got {eps})")


def _param_dtype(dt, *dtypes):
    """What the kernels read the parameters and write their gradients in: the rows' dtype where they all have it, else
    float32."""
    return dt if all(p is None or p == dt for p in dtypes) else torch.float32


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5, residual=None, need_stats=True):
    """``egnn_norm_fwd``: returns ``(y, s, mean, rstd)``; ``s`` is ``x`` itself without a residual, ``mean`` and
    ``rstd`` (rows,) float32 are what :func:`layer_norm_backward` needs, of ``s`` as it is stored (None where
    ``need_stats`` is false)."""
    r = _capi.ext().norm_forward(x, weight, bias, eps, residual, need_stats)
    if r is not None:
        return r
    # a tensor needs a conversion, or an argument is refused
    _check(x, weight, bias, residual, eps)
    if residual is not None and residual.dtype != x.dtype:
        dt = torch.promote_types(x.dtype, residual.dtype)
        _dtype_code(dt)
        x, residual = x.to(dt), residual.to(dt)
    dt, dev, shape = x.dtype, x.device, x.shape
    x2 = _rows(x)
    r2 = None if residual is None else _rows(residual)
    pdt = _param_dtype(dt, *(None if p is None else p.dtype for p in (weight, bias)))
    w, b = _as(weight, pdt), _as(bias, pdt)
    n, c = x2.shape
    y = torch.empty(shape, dtype=dt, device=dev)
    s = x if residual is None else torch.empty(shape, dtype=dt, device=dev)
    stats = torch.empty((2, n), dtype=torch.float32, device=dev) if need_stats else None
    mean, rstd = (stats[0], stats[1]) if need_stats else (None, None)
    check("egnn_norm_fwd",
          _capi.lib().egnn_norm_fwd(EgnnNormDims(n, c, _dtype_code(dt), eps, pdt != dt), x2.data_ptr(), x2.stride(0),
                                    _ptr(r2), 0 if r2 is None else r2.stride(0), _ptr(w), _ptr(b), y.data_ptr(),
                                    None if residual is None else s.data_ptr(), _ptr(mean), _ptr(rstd), _stream(dev)))
    return y, s, mean, rstd


def layer_norm_backward(gy, s, weight, mean, rstd, gsum=None, need_weight=True, need_bias=True, bias_dtype=None):
    """``egnn_norm_bwd``: returns ``(gx, gw, gb)`` from the gradient of ``y`` and, where the sum was used too, of ``s``
    (``gsum``).  ``gx`` is the gradient of x and of the residual; ``gw`` (C,) has the weight's dtype (``s``'s without a
    weight), ``gb`` (C,) has ``bias_dtype`` or that of ``gw``; None where they are not asked for."""
    wdt = s.dtype if weight is None else weight.dtype
    bdt = wdt if bias_dtype is None else bias_dtype
    pdt = _param_dtype(s.dtype, wdt, bdt if need_bias else None)
    r = _capi.ext().norm_backward(gy, s, weight, mean, rstd, gsum, need_weight, need_bias, pdt == torch.float32)
    if r is not None:
        return r[0], _as(r[1], wdt), _as(r[2], bdt)
    dt, dev, shape = s.dtype, s.device, s.shape
    if not s.is_cuda:
        raise RuntimeError("s must be a ROCm device tensor: the layer norm has no CPU path")
    _check(s, weight, None, gsum, 0.0)
    s2 = _rows(s)
    n, c = s2.shape
    if gy.shape != shape or gy.device != dev:
        raise ValueError(f"gy must have the shape {tuple(shape)} (got {tuple(gy.shape)}) and device of s")
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous() or t.device != dev:
            raise ValueError(f"{name} must be the forward's ({n},) float32 statistics")
    g2 = _rows(gy if gy.dtype == dt else gy.to(dt))
    e2 = None if gsum is None else _rows(gsum if gsum.dtype == dt else gsum.to(dt))
    w = _as(weight, pdt)
    gx = torch.empty(shape, dtype=dt, device=dev)
    gw = torch.empty((c,), dtype=pdt, device=dev) if need_weight else None
    gb = torch.empty((c,), dtype=pdt, device=dev) if need_bias else None
    d = EgnnNormDims(n, c, _dtype_code(dt), 0.0, pdt != dt)
    L = _capi.lib()
    nbytes = L.egnn_norm_bwd_workspace_bytes(d) if need_weight or need_bias else 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    check("egnn_norm_bwd",
          L.egnn_norm_bwd(d, g2.data_ptr(), g2.stride(0), s2.data_ptr(), s2.stride(0), _ptr(w), mean.data_ptr(),
                          rstd.data_ptr(), _ptr(e2), 0 if e2 is None else e2.stride(0), gx.data_ptr(), _ptr(gw),
                          _ptr(gb), _ptr(ws), nbytes, _stream(dev)))
    return gx, _as(gw, wdt), _as(gb, bdt)


class LayerNormFn(torch.autograd.Function):
    """``y = LayerNormFn.apply(x, weight, bias, eps, None)`` or ``y, s = LayerNormFn.apply(x, weight, bias, eps,
    residual)``; weight and bias may be None."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, residual):
        y, s, mean, rstd = layer_norm_forward(x, weight, bias, eps, residual)
        ctx.save_for_backward(s, weight, mean, rstd)
        ctx.has_b, ctx.bdt = bias is not None, None if bias is None else bias.dtype
        ctx.xdt, ctx.rdt = x.dtype, None if residual is None else residual.dtype
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, s)

    @staticmethod
    def backward(ctx, gy, gsum=None):
        s, weight, mean, rstd = ctx.saved_tensors
        if gy is None:   # only the sum was used
            gx, gw, gb = gsum, None, None
        else:
            grads = layer_norm_backward(gy, s, weight, mean, rstd, gsum, weight is not None, ctx.has_b,
                                        bias_dtype=ctx.bdt)
            gx, gw, gb = _first_order(grads, gy, gsum, s, weight)
        to = lambda t, dt: t if t is None or t.dtype == dt else t.to(dt)  # noqa: E731
        return to(gx, ctx.xdt), gw, gb, None, None if ctx.rdt is None else to(gx, ctx.rdt)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, residual: Optional[torch.Tensor] = None):
    """``y``, or ``(y, x + residual)`` with a residual (module docstring).  Differentiable in x, weight, bias and
    residual."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return LayerNormFn.apply(x, weight, bias, eps, residual)
    r = _capi.ext().norm_forward(x, weight, bias, eps, residual, False)
    if r is None:   # a tensor needs a conversion, or the call has to be recorded
        if _recorded(x, weight, bias, residual):
            return LayerNormFn.apply(x, weight, bias, eps, residual)
        r = layer_norm_forward(x, weight, bias, eps, residual, need_stats=False)
    return r[0] if residual is None else (r[0], r[1])


def _low_dtype(param_dtype):
    return torch.int16 if param_dtype == torch.float32 else torch.int8


def layer_norm_dropout_forward(x, residual, drop, weight=None, bias=None, eps=1e-5, need_stats=True):
    """``egnn_norm_drop_fwd`` of ``s = residual + dropout(x)``, ``drop`` a :class:`pymolecular_amd.dropout.Dropout`:
    returns ``(y, s, mean, rstd)`` as :func:`layer_norm_forward` does, but that the last one is a pair ``(rstd, low)``
    where ``s`` is bfloat16: what its rounding lost (opaque; int16 beside float32 parameters, else int8), without which
    the gradients would be off by up to 2^-8."""
    r = _capi.ext().norm_drop_forward(x, residual, *drop, weight, bias, eps, need_stats)
    if r is not None:
        return r
    # a tensor needs a conversion, or an argument is refused
    from .dropout import check_drop
    if residual is None:
        raise ValueError("layer_norm_dropout needs the residual: dropout of x alone is pymolecular_amd.dropout")
    _check(x, weight, bias, residual, eps)
    d = check_drop(drop, x.device)
    if residual.dtype != x.dtype:
        dt = torch.promote_types(x.dtype, residual.dtype)
        _dtype_code(dt)
        x, residual = x.to(dt), residual.to(dt)
    dt, dev, shape = x.dtype, x.device, x.shape
    x2, r2 = _rows(x), _rows(residual)
    pdt = _param_dtype(dt, *(None if p is None else p.dtype for p in (weight, bias)))
    w, b = _as(weight, pdt), _as(bias, pdt)
    n, c = x2.shape
    y, s = (torch.empty(shape, dtype=dt, device=dev) for _ in range(2))
    stats = torch.empty((2, n), dtype=torch.float32, device=dev) if need_stats else None
    mean, rstd = (stats[0], stats[1]) if need_stats else (None, None)
    low = torch.empty(shape, dtype=_low_dtype(pdt), device=dev) if need_stats and dt == torch.bfloat16 else None
    with torch.cuda.device(dev):
        check("egnn_norm_drop_fwd",
              _capi.lib().egnn_norm_drop_fwd(EgnnNormDims(n, c, _dtype_code(dt), eps, pdt != dt), d, x2.data_ptr(), x2.stride(0),
                                             r2.data_ptr(), r2.stride(0), _ptr(w), _ptr(b), y.data_ptr(), s.data_ptr(),
                                             _ptr(low), _ptr(mean), _ptr(rstd), _stream(dev)))
    return y, s, mean, rstd if low is None else (rstd, low)


def layer_norm_dropout_backward(gy, s, drop, weight, mean, rstd, gsum=None, need_weight=True, need_bias=True, bias_dtype=None):
    """``egnn_norm_drop_bwd``: returns ``(gx, gresidual, gw, gb)``; arguments and dtypes as in
    :func:`layer_norm_backward`."""
    wdt = s.dtype if weight is None else weight.dtype
    bdt = wdt if bias_dtype is None else bias_dtype
    pdt = _param_dtype(s.dtype, wdt, bdt if need_bias else None)
    rstd, low = rstd if isinstance(rstd, tuple) else (rstd, None)
    if low is not None and low.dtype == torch.int16:   # (the forward had a float32 bias alone)
        pdt = torch.float32
    r = _capi.ext().norm_drop_backward(gy, s, *drop, weight, mean, rstd, low, gsum, need_weight, need_bias, pdt == torch.float32)
    if r is not None:
        return r[0], r[1], _as(r[2], wdt), _as(r[3], bdt)
    from .dropout import check_drop
    dt, dev, shape = s.dtype, s.device, s.shape
    _check(s, weight, None, gsum, 0.0)
    d = check_drop(drop, dev)
    s2 = _rows(s)
    n, c = s2.shape
    if gy.shape != shape or gy.device != dev:
        raise ValueError(f"gy must have the shape {tuple(shape)} (got {tuple(gy.shape)}) and device of s")
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous() or t.device != dev:
            raise ValueError(f"{name} must be the forward's ({n},) float32 statistics")
    if low is not None and (dt != torch.bfloat16 or low.dtype != _low_dtype(pdt) or low.shape != shape or not low.is_contiguous()
                            or low.device != dev):
        raise ValueError("rstd must be what the forward returned with s")
    g2 = _rows(gy if gy.dtype == dt else gy.to(dt))
    e2 = None if gsum is None else _rows(gsum if gsum.dtype == dt else gsum.to(dt))
    w = _as(weight, pdt)
    gx, gr = (torch.empty(shape, dtype=dt, device=dev) for _ in range(2))
    gw = torch.empty((c,), dtype=pdt, device=dev) if need_weight else None
    gb = torch.empty((c,), dtype=pdt, device=dev) if need_bias else None
    nd = EgnnNormDims(n, c, _dtype_code(dt), 0.0, pdt != dt)
    L = _capi.lib()
    nbytes = L.egnn_norm_bwd_workspace_bytes(nd) if need_weight or need_bias else 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    with torch.cuda.device(dev):
        check("egnn_norm_drop_bwd",
              L.egnn_norm_drop_bwd(nd, d, g2.data_ptr(), g2.stride(0), s2.data_ptr(), s2.stride(0), _ptr(low), _ptr(w), mean.data_ptr(),
                                   rstd.data_ptr(), _ptr(e2), 0 if e2 is None else e2.stride(0), gx.data_ptr(), gr.data_ptr(),
                                   _ptr(gw), _ptr(gb), _ptr(ws), nbytes, _stream(dev)))
    return gx, gr, _as(gw, wdt), _as(gb, bdt)


class LayerNormDropoutFn(torch.autograd.Function):
    """``y, s = LayerNormDropoutFn.apply(x, residual, p, rng, site, weight, bias, eps)``; weight and bias may be None."""

    @staticmethod
    def forward(ctx, x, residual, p, rng, site, weight, bias, eps):
        y, s, mean, rstd = layer_norm_dropout_forward(x, residual, (p, rng, site), weight, bias, eps)
        rstd, low = rstd if isinstance(rstd, tuple) else (rstd, None)
        ctx.save_for_backward(s, weight, mean, rstd, low, rng)
        ctx.p, ctx.site = p, site
        ctx.has_b, ctx.bdt = bias is not None, None if bias is None else bias.dtype
        ctx.xdt, ctx.rdt = x.dtype, residual.dtype
        ctx.set_materialize_grads(False)
        return y, s

    @staticmethod
    def backward(ctx, gy, gsum=None):
        s, weight, mean, rstd, low, rng = ctx.saved_tensors
        rstd = rstd if low is None else (rstd, low)
        drop = (ctx.p, rng, ctx.site)
        if gy is None:   # only the sum was used, if anything was
            if gsum is None:
                return (None,) * 8
            from .dropout import dropout
            gx, gr, gw, gb = dropout(gsum, ctx.p, rng, site=ctx.site), gsum, None, None
        else:
            grads = layer_norm_dropout_backward(gy, s, drop, weight, mean, rstd, gsum, weight is not None, ctx.has_b,
                                                bias_dtype=ctx.bdt)
            gx, gr, gw, gb = _first_order(grads, gy, gsum, s, weight)
        to = lambda t, dt: t if t.dtype == dt else t.to(dt)  # noqa: E731
        return to(gx, ctx.xdt), to(gr, ctx.rdt), None, None, None, gw, gb, None


def layer_norm_dropout(x: torch.Tensor, residual: torch.Tensor, drop, weight: Optional[torch.Tensor] = None,
                       bias: Optional[torch.Tensor] = None, eps: float = 1e-5):
    """``(y, s)`` with ``s = residual + dropout(x)`` and ``y`` its norm; ``drop`` is a
    :class:`pymolecular_amd.dropout.Dropout`.  Differentiable in x, residual, weight and bias."""
    tensors = (x, residual, weight, bias)
    if (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)) or _recorded(*tensors):
        return LayerNormDropoutFn.apply(x, residual, *drop, weight, bias, eps)
    return layer_norm_dropout_forward(x, residual, drop, weight, bias, eps, need_stats=False)[:2]
