"""Norm of heads and rotation by position in float64 on the CPU (numpy): pairs as complex numbers, angles in extended
precision."""
from __future__ import annotations

import numpy as np

__all__ = ["turns_ref", "qk_norm_rotary_ref", "qk_norm_rotary_grads_ref"]


def _split(x, rotary, interleaved):
    """(complex pairs of the first values, the rest)."""
    if interleaved:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
    else:
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
    return a + 1j * b, x[..., rotary:]


def _join(z, rest, interleaved):
    if interleaved:
        ab = np.stack([z.real, z.imag], axis=-1).reshape(*z.shape[:-1], -1)
    else:
        ab = np.concatenate([z.real, z.imag], axis=-1)
    return np.concatenate([ab, rest], axis=-1)


def turns_ref(positions, base, rotary):
    """e^(i position frequency), (N, 1, rotary / 2)."""
    f = np.longdouble(base) ** (-2 * np.arange(rotary // 2, dtype=np.longdouble) / max(rotary, 1))
    a = np.remainder(np.asarray(positions, dtype=np.int64).astype(np.longdouble)[:, None, None] * f,
                     2 * np.longdouble("3.14159265358979323846264338327950288"))
    return np.exp(1j * a.astype(np.float64))


def _norm(x, eps):
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return r, x * r


def qk_norm_rotary_ref(x, w, positions, base=10000.0, rotary=None, interleaved=False, eps=1e-6):
    """x (N, heads, d), w (d,) or None."""
    rotary = x.shape[-1] if rotary is None else rotary
    _, y = _norm(x, eps)
    y = y if w is None else y * w
    z, rest = _split(y, rotary, interleaved)
    return _join(z * turns_ref(positions, base, rotary) if rotary else z, rest, interleaved)


def qk_norm_rotary_grads_ref(g, x, w, positions, base=10000.0, rotary=None, interleaved=False, eps=1e-6):
    """(gx, gw)."""
    rotary = x.shape[-1] if rotary is None else rotary
    r, xh = _norm(x, eps)
    z, rest = _split(g, rotary, interleaved)
    gn = _join(z * np.conj(turns_ref(positions, base, rotary)) if rotary else z, rest, interleaved)
    t = gn if w is None else gn * w
    return r * (t - xh * (t * xh).mean(-1, keepdims=True)), (gn * xh).sum((0, 1))
