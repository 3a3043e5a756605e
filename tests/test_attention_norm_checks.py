"""Segment attention and layer norm without a GPU: the float64 oracle's own gradients, and what the C entries refuse
before they touch the device."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import attention_ref as ref
from pymolecular_amd import _capi

BUF = 1 << 12   # a non-NULL aligned stand-in address, never dereferenced by the calls below


def _inputs():
    r = np.random.Generator(np.random.PCG64(0))
    q, k, v, go = r.standard_normal((12, 4, 6)), r.standard_normal((15, 2, 6)), r.standard_normal((15, 2, 6)), r.standard_normal((12, 4, 6))
    return r, q, k, v, go, ([0, 5, 5, 9, 11], [0, 4, 7, 7, 13], r.random(15) < 0.8)


def test_oracle_gradients_against_differences_and_autograd():
    r, q, k, v, go, seg = _inputs()
    grads = ref.segment_attention_grads_ref(go, q, k, v, *seg, scale=0.7)
    f = lambda *a: (ref.segment_attention_ref(*a, *seg, scale=0.7)[0] * go).sum()  # noqa: E731
    for i, g in enumerate(grads):
        u = r.standard_normal(g.shape)
        at = lambda t: [x + t * u if j == i else x for j, x in enumerate((q, k, v))]  # noqa: E731
        assert abs((f(*at(1e-5)) - f(*at(-1e-5))) / 2e-5 - (g * u).sum()) < 1e-7 * np.abs(g).sum()
    tq, tk, tv = (torch.from_numpy(t).requires_grad_() for t in (q, k, v))
    total = 0
    for b in range(4):
        i = slice(seg[0][b], seg[0][b + 1])
        keep = np.arange(seg[1][b], seg[1][b + 1])
        keep = keep[seg[2][keep]]
        if i.stop > i.start and len(keep):
            kk, vv = (t[keep].repeat_interleave(2, dim=1) for t in (tk, tv))
            p = torch.softmax(0.7 * torch.einsum("ihd,jhd->hij", tq[i], kk), dim=2)
            total = total + (torch.einsum("hij,jhd->ihd", p, vv) * torch.from_numpy(go[i])).sum()
    for a, b in zip(torch.autograd.grad(total, (tq, tk, tv)), grads):
        assert np.allclose(a.numpy(), b, atol=1e-12)


def test_oracle_rows_without_keys():
    _, q, k, v, go, seg = _inputs()
    out, lse = ref.segment_attention_ref(q, k, v, *seg)
    assert not out[5:9].all() and np.isneginf(lse[:, 5:9]).all() and np.isneginf(lse[:, 11:]).all()   # no keys; outside
    assert all(not g[5:9].any() for g in ref.segment_attention_grads_ref(go, q, k, v, *seg)[:1])


def test_oracle_layer_norm_gradients():
    r = np.random.Generator(np.random.PCG64(1))
    x, res, w, b, gy, gs = *(r.standard_normal((7, 9)) for _ in range(2)), r.standard_normal(9), r.standard_normal(9), \
        r.standard_normal((7, 9)), r.standard_normal((7, 9))
    t = [torch.from_numpy(a).requires_grad_() for a in (x, w, b)]
    s = t[0] + torch.from_numpy(res)
    y = torch.nn.functional.layer_norm(s, (9,), t[1], t[2], 1e-5)
    want = torch.autograd.grad((y * torch.from_numpy(gy)).sum() + (s * torch.from_numpy(gs)).sum(), t)
    y_ref, s_ref = ref.layer_norm_ref(x, w, b, 1e-5, res)
    assert np.allclose(y.detach().numpy(), y_ref, atol=1e-12)
    for g, a in zip(ref.layer_norm_grads_ref(gy, s_ref, w, 1e-5, gs), want):
        assert np.allclose(g, a.numpy(), atol=1e-12)


def _attn(**kw):
    d = dict(Nq=100, Nk=100, n_seg=4, Hq=4, Hkv=2, D=32, dtype=1, scale=0.5)
    return _capi.EgnnAttnDims(**{**d, **kw})


def _strides(**kw):
    s = _capi.EgnnAttnStrides(*([256, 64] * 8))
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def _fwd(d, s, ptrs=None, ws=(None, 0)):
    p = [BUF] * 8 if ptrs is None else ptrs
    return _capi.lib().egnn_attn_fwd(d, s, *p[:6], *p[6:8], *ws, None)   # q k v q_ptr kv_ptr mask out lse, workspace, stream


@pytest.mark.parametrize("kw", [dict(Hq=3), dict(Hkv=0), dict(D=12), dict(D=136), dict(D=0), dict(dtype=2), dict(scale=0.0),
                                dict(scale=float("nan")), dict(scale=float("inf")), dict(Nq=-1), dict(Nk=1 << 31),
                                dict(Nq=1 << 30), dict(n_seg=-1)])
def test_attention_dims_refused(kw):
    L = _capi.lib()
    assert _fwd(_attn(**kw), _strides()) == _capi.EGNN_ERR_DIMS
    assert L.egnn_attn_bwd(_attn(**kw), _strides(), *([BUF] * 12), None, 0, None) == _capi.EGNN_ERR_DIMS
    assert L.egnn_attn_fwd_workspace_bytes(_attn(**kw)) == L.egnn_attn_bwd_workspace_bytes(_attn(**kw)) == 0


def test_attention_arguments_refused():
    L = _capi.lib()
    assert L.egnn_attn_fwd(None, None, *([None] * 9), 0, None) == 1
    for i in range(8):
        if i not in (5, 7):                                           # mask and lse may be NULL
            assert _fwd(_attn(), _strides(), [None if j == i else BUF for j in range(8)]) == 1, i
    for i in (0, 1, 2, 6):
        assert _fwd(_attn(), _strides(), [BUF + 8 if j == i else BUF for j in range(8)]) == 4, i
    for kw in (dict(q_row=260), dict(k_head=12), dict(v_row=-256), dict(out_head=24), dict(out_row=16)):
        assert _fwd(_attn(), _strides(**kw)) == 3, kw
    # a single query over a long axis is split: the workspace is asked for and checked
    d = _attn(Nq=1, Nk=100000, n_seg=1)
    need = L.egnn_attn_fwd_workspace_bytes(d)
    assert need > 0 and L.egnn_attn_bwd_workspace_bytes(d) > 0
    assert _fwd(d, _strides()) == 5 and _fwd(d, _strides(), ws=(BUF, need - 1)) == 5 and _fwd(d, _strides(), ws=(BUF + 4, need)) == 4
    # the backward: NULL or misaligned tensors, overlapping gradients, no room for its row sums
    bwd = lambda p, s=_strides(), ws=(BUF, 1 << 40): L.egnn_attn_bwd(_attn(), s, *p, *ws, None)  # noqa: E731
    for i in range(12):                                               # q k v out lse go q_ptr kv_ptr mask gq gk gv
        if i != 8:
            assert bwd([None if j == i else BUF for j in range(12)]) == 1, i
    assert bwd([BUF] * 12, _strides(grad_k_head=16)) == 3 and bwd([BUF + 4 if j == 9 else BUF for j in range(12)]) == 4
    assert bwd([BUF] * 12, ws=(None, 0)) == 5


def test_norm_arguments_refused():
    L = _capi.lib()
    dims = lambda **kw: _capi.EgnnNormDims(**{**dict(N=10, C=64, dtype=0, eps=1e-5), **kw})  # noqa: E731
    fwd = lambda d, x=BUF, ldx=64, r=None, y=BUF, s=None, m=BUF, v=BUF: L.egnn_norm_fwd(d, x, ldx, r, 64, BUF, BUF, y, s, m, v, None)  # noqa: E731
    for kw in (dict(C=0), dict(C=(1 << 20) + 1), dict(N=-1), dict(N=1 << 31), dict(dtype=3), dict(eps=-1.0),
               dict(eps=float("nan")), dict(eps=float("inf"))):
        assert fwd(dims(**kw)) == 2 and L.egnn_norm_bwd_workspace_bytes(dims(**kw)) == 0, kw
    assert fwd(None) == 1 and fwd(dims(), x=None) == 1 and fwd(dims(), y=None) == 1 and fwd(dims(), m=None) == 1
    assert fwd(dims(), r=BUF) == 1                                    # a residual needs the sum's buffer
    assert fwd(dims(), ldx=-64) == 3 and fwd(dims(), x=BUF + 2) == 4
    bwd = lambda d, g=BUF, ws=BUF, nb=1 << 30, gw=BUF: L.egnn_norm_bwd(d, g, 64, BUF, 64, None, BUF, BUF, None, 0, BUF, gw, None, ws, nb, None)  # noqa: E731
    assert bwd(dims(), g=None) == 1 and bwd(dims(), ws=None) == 5 and bwd(dims(), nb=16) == 5 and bwd(dims(C=0)) == 2
    assert bwd(dims(), g=BUF + 1) == 4


def test_no_cpu_path():
    from pymolecular_amd.layer_norm import layer_norm
    from pymolecular_amd.segment_attention import segment_attention
    with pytest.raises(RuntimeError, match="no CPU path"):
        segment_attention(*(torch.zeros(4, 2, 16) for _ in range(3)), torch.tensor([0, 4], dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        layer_norm(torch.zeros(4, 16))


def test_struct_sizes():
    assert ctypes.sizeof(_capi.EgnnAttnDims) == 40 and ctypes.sizeof(_capi.EgnnAttnStrides) == 128
    assert ctypes.sizeof(_capi.EgnnNormDims) == 24
