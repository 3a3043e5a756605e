"""Norm and rotation of heads without a GPU: the oracle's gradients, its rotation, and what the entries refuse before they
touch the device."""
import ctypes

import numpy as np
import pytest
import torch

from oracle.qk_ref import qk_norm_rotary_grads_ref, qk_norm_rotary_ref
from pymolecular_amd import _capi

BUF = 1 << 12   # a non-NULL aligned stand-in address, never dereferenced by the calls below


@pytest.mark.parametrize("rotary,interleaved", [(8, False), (8, True), (4, False), (6, True), (0, False)])
def test_oracle_gradients_against_differences(rotary, interleaved):
    r = np.random.Generator(np.random.PCG64(rotary))
    x, g, u = r.standard_normal((3, 6, 3, 8))
    w, uw = r.standard_normal((2, 8))
    pos = np.array([0, 5, -7, 1000, 3, 2 ** 31])
    how = (pos, 100.0, rotary, interleaved, 1e-3)
    f = lambda a, b: (qk_norm_rotary_ref(a, b, *how) * g).sum()  # noqa: E731
    gx, gw = qk_norm_rotary_grads_ref(g, x, w, *how)
    h = 1e-5
    assert abs((f(x + h * u, w) - f(x - h * u, w)) / (2 * h) - (gx * u).sum()) < 1e-7
    assert abs((f(x, w + h * uw) - f(x, w - h * uw)) / (2 * h) - (gw * uw).sum()) < 1e-7


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_products_depend_on_distances(interleaved):
    r = np.random.Generator(np.random.PCG64(1))
    q, k = r.standard_normal((2, 1, 1, 16))
    at = lambda x, p: qk_norm_rotary_ref(x, None, np.array([p]), 50.0, 12, interleaved)[0, 0]  # noqa: E731
    want = at(q, 7) @ at(k, 0)
    # an angle near p carries the product's and the frequency's rounding to 64 bits, 2^-63 p, in the query and in the key; it
    # moves the product of heads of length 4 by at most 16 times that
    for p in (1, 100, 2 ** 30):
        assert abs(at(q, p + 7) @ at(k, p) - want) < 1e-12 + 2 * 16 * p * 2.0 ** -63
    # the definition, by real numbers
    c, s, y = np.cos(3.0), np.sin(3.0), q[0, 0] / np.sqrt((q * q).mean() + 1e-6)
    a, b = (0, 1) if interleaved else (0, 6)
    assert np.allclose(at(q, 3)[[a, b]], [y[a] * c - y[b] * s, y[b] * c + y[a] * s]) and np.allclose(at(q, 3)[12:], y[12:])


def _dims(**kw):
    return _capi.EgnnQkDims(**{**dict(N=10, Hq=4, Hk=2, D=32, rotary=32, interleaved=0, dtype=1, f32_params=0, index64=0, eps=1e-6,
                                      base=1e4), **kw})


def _strides(**kw):
    s = _capi.EgnnQkStrides(*([256, 32] * 8))
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def test_arguments_refused():
    L = _capi.lib()
    fwd = lambda d=None, s=None, p=None: L.egnn_qk_fwd(d or _dims(), s or _strides(), *(p or [BUF] * 7), None)  # noqa: E731
    bwd = lambda d=None, s=None, p=None, ws=(BUF, 1 << 40): L.egnn_qk_bwd(d or _dims(), s or _strides(), *(p or [BUF] * 11), *ws, None)  # noqa: E731
    for kw in (dict(N=-1), dict(N=1 << 31), dict(Hq=0), dict(Hk=0), dict(Hq=4097), dict(D=31), dict(D=0), dict(D=130),
               dict(rotary=-2), dict(rotary=34), dict(rotary=7), dict(interleaved=2), dict(dtype=2), dict(f32_params=2),
               dict(index64=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(base=0.5), dict(base=float("inf")),
               dict(base=float("nan"))):
        assert fwd(_dims(**kw)) == bwd(_dims(**kw)) == 2 and L.egnn_qk_bwd_workspace_bytes(_dims(**kw)) == 0, kw
    one = lambda n, i, v=None: [v if j == i else BUF for j in range(n)]  # noqa: E731
    for i in (0, 1, 4, 5, 6):                 # q k qw kw pos q_out k_out
        assert fwd(p=one(7, i)) == 1, i
    for i in (0, 1, 2, 3, 6, 7, 8):           # gq gk q k qw kw pos gq gk gqw gkw
        assert bwd(p=one(11, i)) == 1, i
    assert L.egnn_qk_fwd(None, _strides(), *([BUF] * 7), None) == 1 == L.egnn_qk_fwd(_dims(), None, *([BUF] * 7), None)
    for kw in (dict(q_row=-1), dict(k_head=-1), dict(q_out_head=31), dict(k_out_row=63), dict(q_out_row=127)):
        assert fwd(s=_strides(**kw)) == 3, kw
    for kw in (dict(k_row=-1), dict(grad_q_out_row=-1), dict(grad_k_head=31), dict(grad_q_row=127)):
        assert bwd(s=_strides(**kw)) == 3, kw
    for i in range(7):
        assert fwd(p=one(7, i, BUF + 1)) == 4, i
    for i in range(11):
        assert bwd(p=one(11, i, BUF + 1)) == 4, i
    need = L.egnn_qk_bwd_workspace_bytes(_dims())
    assert need > 0 and bwd(ws=(None, 0)) == bwd(ws=(BUF, need - 1)) == 5 and bwd(ws=(BUF + 8, need)) == 4


def test_python_refusals():
    from pymolecular_amd.qk_norm_rotary import qk_norm_rotary, qk_norm_rotary_attention
    q = torch.zeros(4, 2, 16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        qk_norm_rotary(q, q)
    with pytest.raises(RuntimeError, match="no CPU path"):
        qk_norm_rotary_attention(q.repeat(1, 3, 1), 2, torch.tensor([0, 4], dtype=torch.int32))


def test_struct_sizes():
    assert ctypes.sizeof(_capi.EgnnQkDims) == 56 and ctypes.sizeof(_capi.EgnnQkStrides) == 128
