"""Dropout without a GPU: the oracle's generator, its statistics, and what the C entries refuse before they touch the
device."""
import ctypes

import numpy as np
import pytest
import torch

from oracle.dropout_ref import dropout_grad_ref, dropout_ref, keep_ref, philox
from pymolecular_amd import _capi

BUF = 1 << 12   # a non-NULL aligned stand-in address, never dereferenced by the calls below


def test_generator_known_answers():
    # the published answers for a counter and a key of zeros, with 7 and with 10 rounds
    assert [int(x) for x in philox((0,) * 4, (0,) * 2)] == [0x5f6fb709, 0x0d893f64, 0x4f121f81, 0x4f730a48]
    assert [int(x) for x in philox((0,) * 4, (0,) * 2, 10)] == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]


@pytest.mark.parametrize("p", [0.05, 0.1, 0.5])
def test_shares_and_independence(p):
    n, c = 2000, 259
    keep, up = keep_ref(n, c, p, 1234567890123, 7)
    q = 1 - round(65536 * p) / 65536
    assert up == 1 / q
    sigma = np.sqrt(q * (1 - q))
    assert abs(keep.mean() - q) < 5 * sigma / np.sqrt(n * c)
    # columns and rows: the largest of so many deviations is below 6 sigma but for 1e-6; neighbours do not correlate
    assert np.abs(keep.mean(0) - q).max() < 6 * sigma / np.sqrt(n) and np.abs(keep.mean(1) - q).max() < 6 * sigma / np.sqrt(c)
    z = (keep - q) / sigma
    for a, b in ((z[:, 1:], z[:, :-1]), (z[1:], z[:-1])):
        assert abs((a * b).mean()) < 5 / np.sqrt(a.size)
    for other in (keep_ref(n, c, p, 1234567890124, 7), keep_ref(n, c, p, 1234567890123, 8)):
        assert abs((z * ((other[0] - q) / sigma)).mean()) < 5 / np.sqrt(n * c)
    assert np.array_equal(keep_ref(50, c, p, 1234567890123, 7, row0=40)[0], keep[40:90])


def test_oracle_gradient_against_differences():
    r = np.random.Generator(np.random.PCG64(0))
    x, gy, u = r.standard_normal((3, 9, 20))
    g = dropout_grad_ref(gy, 0.3, -5, 2 ** 40)
    f = lambda t: (dropout_ref(t, 0.3, -5, 2 ** 40, x) * gy).sum()  # noqa: E731
    assert abs((f(x + 1e-3 * u) - f(x - 1e-3 * u)) / 2e-3 - (g * u).sum()) < 1e-9


def test_ends_of_the_range():
    assert keep_ref(4, 9, 0.0, 1, 2)[0].all() and keep_ref(4, 9, 0.0, 1, 2)[1] == 1.0
    assert not keep_ref(4, 9, 1.0, 1, 2)[0].any()


def _drop(p=0.1, rng=BUF):
    return _capi.EgnnDropout(rng, 0, p)


def test_dropout_arguments_refused():
    L = _capi.lib()
    f = lambda d=None, dt=0, n=10, c=64, x=BUF, ldx=64, r=None, ldr=64, y=BUF: L.egnn_dropout(d or _drop(), dt, n, c, x, ldx, r, ldr, y, None)  # noqa: E731
    assert L.egnn_dropout(None, 0, 10, 64, BUF, 64, None, 0, BUF, None) == 1
    for kw in (dict(dt=2), dict(n=-1), dict(n=1 << 31), dict(c=0), dict(c=(1 << 20) + 1), dict(d=_drop(p=-0.1)),
               dict(d=_drop(p=1.1)), dict(d=_drop(p=float("nan")))):
        assert f(**kw) == _capi.EGNN_ERR_DIMS, kw
    assert f(x=None) == f(y=None) == f(d=_drop(rng=None)) == 1
    assert f(ldx=-1) == f(r=BUF, ldr=-1) == 3
    assert f(x=BUF + 2) == f(y=BUF + 2) == f(r=BUF + 1) == f(d=_drop(rng=BUF + 4)) == 4
    assert f(n=0, x=None, y=None) == 0


def test_norm_with_dropout_arguments_refused():
    L = _capi.lib()
    dims = lambda **kw: _capi.EgnnNormDims(**{**dict(N=10, C=64, dtype=0, eps=1e-5), **kw})  # noqa: E731
    fwd = lambda d=None, dr=None, x=BUF, r=BUF, y=BUF, s=BUF, m=BUF, v=BUF, ldr=64, w=BUF, low=None: L.egnn_norm_drop_fwd(  # noqa: E731
        d or dims(), dr or _drop(), x, 64, r, ldr, w, BUF, y, s, low, m, v, None)
    for d in (dims(C=0), dims(N=1 << 31), dims(eps=-1.0), dims(dtype=5), dims(f32_params=2)):
        assert fwd(d) == 2
    assert fwd(dr=_drop(p=2.0)) == 2
    for kw in (dict(x=None), dict(r=None), dict(y=None), dict(s=None), dict(m=None), dict(dr=_drop(rng=None))):
        assert fwd(**kw) == 1, kw
    assert fwd(ldr=-4) == 3 and fwd(r=BUF + 2) == fwd(s=BUF + 2) == fwd(w=BUF + 2) == fwd(dr=_drop(rng=BUF + 4)) == 4
    bwd = lambda d=None, dr=None, g=BUF, gx=BUF, gr=BUF, ws=BUF, nb=1 << 30, ldgs=0, low=None: L.egnn_norm_drop_bwd(  # noqa: E731
        d or dims(), dr or _drop(), g, 64, BUF, 64, low, None, BUF, BUF, BUF, ldgs, gx, gr, BUF, None, ws, nb, None)
    assert bwd(dims(C=0)) == bwd(dr=_drop(p=-1.0)) == 2 and bwd(g=None) == bwd(gx=None) == bwd(gr=None) == 1
    assert fwd(low=BUF) == bwd(low=BUF) == 2   # beside float32 rows
    assert fwd(dims(dtype=1, f32_params=1), low=BUF + 1) == bwd(dims(dtype=1, f32_params=1), low=BUF + 1) == 4
    assert bwd(ldgs=-1) == 3 and bwd(gr=BUF + 2) == 4 and bwd(ws=None) == bwd(nb=16) == 5
    assert L.egnn_norm_drop_fwd(dims(), None, *([BUF, 64] * 2), *([BUF] * 7), None) == 1


def test_python_refusals():
    from pymolecular_amd.dropout import Dropout, check_drop, dropout
    from pymolecular_amd.layer_norm import layer_norm_dropout
    rng = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        dropout(torch.zeros(4, 16), 0.1, rng)
    with pytest.raises(RuntimeError, match="no CPU path"):
        layer_norm_dropout(torch.zeros(4, 16), torch.zeros(4, 16), Dropout(0.1, rng))
    with pytest.raises(ValueError, match="needs the residual"):
        layer_norm_dropout(torch.zeros(4, 16), None, Dropout(0.1, rng))
    cpu = torch.device("cpu")
    assert check_drop(Dropout(0.25, rng, 3), cpu).site == 3
    for bad in (Dropout(-0.1, rng), Dropout(float("nan"), rng), Dropout(1.5, rng), Dropout(0.1, rng.int()),
                Dropout(0.1, rng[:1]), Dropout(0.1, torch.zeros(4, dtype=torch.int64)[::2])):
        with pytest.raises(ValueError):
            check_drop(bad, cpu)
    with pytest.raises(ValueError):
        check_drop(Dropout(0.1, rng), torch.device("cuda", 0))


def test_struct_size():
    assert ctypes.sizeof(_capi.EgnnDropout) == 24
