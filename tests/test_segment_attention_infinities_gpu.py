"""Segment attention where rows that take part hold infinities: what the padding of tiles does must not show.

The float64 formulas say which results are finite, infinite and NaN; those places have to be the same, and the finite
values within the bounds of test_segment_attention_gpu.py (1e-5 in float32, 2^-7 in bfloat16).
"""
import numpy as np
import pytest
import torch

from oracle import attention_ref as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
INF = float("inf")
# lq, lk, heads, kv_heads, d: small segments, tiles of a wave (alone and among small ones), of 64 and 128 rows, parts
SHAPES = [([20, 7, 31], None, 4, 2, 32), ([20, 7, 31], None, 4, 4, 64), ([20] * 8 + [40], None, 2, 2, 16),
          ([8] * 30 + [40], [20] * 30 + [90], 4, 4, 32), ([20, 9], None, 2, 1, 128), ([80, 33], None, 2, 2, 64),
          ([2100], None, 1, 1, 32), ([2], [3000], 2, 1, 64)]


def _np(t):
    return t.detach().double().cpu().numpy()


def _case(lq, lk, hq, hk, d, dtype):
    gen = torch.Generator().manual_seed(1)
    rand = lambda *s: torch.randn(s, generator=gen).to(dtype).cuda()  # noqa: E731
    off = lambda n: torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32, device="cuda")  # noqa: E731
    nq, nk = sum(lq), sum(lk or lq)
    q_ptr = off(lq)
    return rand(nq, hq, d), rand(nk, hk, d), rand(nk, hk, d), rand(nq, hq, d), q_ptr, off(lk) if lk else q_ptr


def _compare(q, k, v, go, q_ptr, kv_ptr, names):
    from pymolecular_amd.segment_attention import segment_attention_backward, segment_attention_forward
    out, lse = segment_attention_forward(q, k, v, q_ptr, kv_ptr)
    got = dict(zip(("out", "dq", "dk", "dv"), (out, *segment_attention_backward(go, q, k, v, out, lse, q_ptr, kv_ptr))))
    a, ptrs = [_np(t) for t in (q, k, v)], (q_ptr.cpu().numpy(), kv_ptr.cpu().numpy())
    with np.errstate(all="ignore"):
        want = dict(zip(("out", "dq", "dk", "dv"), (ref.segment_attention_ref(*a, *ptrs)[0],
                                                    *ref.segment_attention_grads_ref(_np(go), *a, *ptrs))))
    for n in names:
        x, y = _np(got[n]), want[n]
        for kind in (np.isnan, np.isposinf, np.isneginf):
            assert np.array_equal(kind(x), kind(y)), (n, kind.__name__)
        ok = np.isfinite(y)
        assert np.linalg.norm((x - y)[ok]) <= (1e-5 if q.dtype == F32 else 2.0 ** -7) * np.linalg.norm(y[ok]), n


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_broadcast_rows(shape, dtype):
    # every row is one row in memory, which holds an infinity: each output has it, not 0 times it
    q, k, v, go, a, b = _case(*shape, dtype)
    v[0, :, 5] = INF
    _compare(q, k, v[:1].expand(v.shape), go, a, b, ["out"])
    q, k, v, go, a, b = _case(*shape, dtype)
    go[0, :, 2] = -INF
    _compare(q, k, v, go[:1].expand(go.shape), a, b, ["out", "dv"])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_an_infinite_key(shape, dtype):
    # all scores of a key are -inf: no probability, no gradient of it, and the other keys' are finite; dq is 0 times an
    # infinity in that feature
    q, k, v, go, a, b = _case(*shape, dtype)
    k[3, 0, 2] = -INF
    _compare(q.abs(), k, v, go, a, b, ["out", "dq", "dk", "dv"])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_infinite_values(shape, dtype):
    # an infinity of a value reaches the segment's outputs in its feature; dv, made without it, stays finite
    q, k, v, go, a, b = _case(*shape, dtype)
    v[3, 0, 5], v[2, 0, 1] = INF, -INF
    _compare(q, k, v, go, a, b, ["out", "dv"])
