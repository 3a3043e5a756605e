"""The embedding without a GPU: the oracle's gradient, and what the entries refuse before they touch the device."""
import ctypes

import numpy as np
import pytest
import torch

from oracle.embedding_ref import embedding_grad_ref, embedding_ref
from pymolecular_amd import _capi

BUF = 1 << 12   # a non-NULL aligned stand-in address, never dereferenced by the calls below


def test_oracle_gradient_against_differences():
    r = np.random.Generator(np.random.PCG64(0))
    t = np.array([3, 0, 3, -1, 6, 2, 3, 9])
    w, u, go = r.standard_normal((7, 5)), r.standard_normal((7, 5)), r.standard_normal((8, 5))
    f = lambda x: (embedding_ref(t, x, 1.5) * go).sum()  # noqa: E731
    g = embedding_grad_ref(go, t, 7, 1.5)
    assert abs((f(w + u) - f(w - u)) / 2 - (g * u).sum()) < 1e-12
    assert not embedding_grad_ref(go, t, 7, 1.5, padding=3)[3].any()
    assert not embedding_ref(t, w)[[3, 7]].any()


def _dims(**kw):
    return _capi.EgnnEmbedDims(**{**dict(N=10, V=20, C=64, dtype=0, f32_table=0, index64=1, scale=1.0), **kw})


def test_arguments_refused():
    L = _capi.lib()
    fwd = lambda d=None, t=BUF, w=BUF, ldw=64, o=BUF: L.egnn_embed_fwd(d or _dims(), t, w, ldw, o, None)  # noqa: E731
    bwd = lambda d=None, pad=-1, g=BUF, ldg=64, t=BUF, gw=BUF, ws=BUF, nb=1 << 50: L.egnn_embed_bwd(  # noqa: E731
        d or _dims(), pad, g, ldg, t, gw, ws, nb, None)
    for kw in (dict(N=-1), dict(N=1 << 31), dict(V=0), dict(V=-3), dict(C=0), dict(C=(1 << 20) + 1), dict(dtype=2),
               dict(f32_table=2), dict(index64=-1), dict(scale=float("inf")), dict(scale=float("nan")),
               dict(V=(1 << 31) - 1, C=1 << 10)):
        assert fwd(_dims(**kw)) == bwd(_dims(**kw)) == 2 and L.egnn_embed_bwd_workspace_bytes(_dims(**kw)) == 0, kw
    assert L.egnn_embed_fwd(None, BUF, BUF, 64, BUF, None) == 1 == L.egnn_embed_bwd(None, -1, BUF, 64, BUF, BUF, None, 0, None)
    assert fwd(t=None) == fwd(w=None) == fwd(o=None) == bwd(g=None) == bwd(t=None) == bwd(gw=None) == 1
    assert fwd(ldw=-1) == bwd(ldg=-1) == 3
    assert fwd(t=BUF + 4) == fwd(w=BUF + 2) == fwd(o=BUF + 1) == bwd(g=BUF + 2) == bwd(gw=BUF + 2) == bwd(ws=BUF + 8) == 4
    assert bwd(_dims(dtype=1, f32_table=1), gw=BUF + 2) == 4
    assert bwd(pad=20) == bwd(pad=-2) == 2
    assert fwd(_dims(N=0), t=None, w=None, o=None) == 0
    # forms that need a workspace say so: partial tables, and the whole order sorted
    for d in (_dims(N=100000, V=50), _dims(N=100000, V=50000)):
        need = L.egnn_embed_bwd_workspace_bytes(d)
        assert need > 0 and bwd(d, ws=None) == bwd(d, nb=need - 1) == 5


@pytest.mark.parametrize("v", [1, 2, 119, 1024, 4096, 4097, 131072, 1 << 24, (1 << 31) - 1])
@pytest.mark.parametrize("n", [0, 1, 4096, 4097, 6145, 1 << 17, (1 << 31) - 1])
@pytest.mark.parametrize("c", [1, 128, 259])
def test_workspaces_of_every_size(n, v, c):
    # at most 16 bytes a token, twice, and as many bytes as grad_out holds in fp32
    need = _capi.lib().egnn_embed_bwd_workspace_bytes(_dims(N=n, V=v, C=c))
    assert 0 <= need <= 17 * n + 4 * n * c + (1 << 20) * 8


def test_python_refusals():
    from pymolecular_amd.embedding import embedding, embedding_backward
    w, t = torch.zeros(4, 16), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        embedding(t, w)
    with pytest.raises(RuntimeError, match="no CPU path"):
        embedding_backward(torch.zeros(3, 16), t, 4)
    for padding in (-1, 4):
        with pytest.raises(ValueError, match="padding"):
            embedding(t, w, padding=padding)
    with pytest.raises(ValueError, match="weight must be"):
        embedding(t, w[0])
    with pytest.raises(ValueError, match="grad_out must be"):
        embedding_backward(torch.zeros(2, 16), t, 4)


def test_struct_size():
    assert ctypes.sizeof(_capi.EgnnEmbedDims) == 32
