"""Segment attention's gradients where keys and values have a common part, as a projection's bias gives them.

A constant added to all keys changes no probability, so it must not reach dq beyond rounding.  With c times the spread in
both, bfloat16: every ds is rounded once, 2^-9 at most, and what the roundings leave of sum_j ds_j = 0 meets keys of size
sqrt(1 + c^2) times their spread; the result is rounded too: 2 x 2^-9 (1 + sqrt(1 + c^2)) of dq's norm.  dk and dv do not see
the common part: 4 x 2^-9, as without it.  float32: 1e-5 times (1 + c^2), as delta is a product of do and o, which both
have the factor's share.
"""
import numpy as np
import pytest
import torch

from oracle import attention_ref as ref
from test_segment_attention_gpu import _case, _np, _rel

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
# small segments; longer ones among them; waves, 64 rows, 128 rows, parts
SHAPES = [([9, 29, 17, 1, 2, 31], None, 4, 4, 32), ([12, 40, 20, 36, 9, 55] * 4, None, 4, 4, 32), ([10, 40] * 5, None, 4, 2, 16),
          ([4, 30, 17, 22], [700, 100, 300, 900], 4, 4, 32), ([9, 20, 33], [500, 800, 60], 4, 1, 72), ([80, 64, 33], None, 2, 2, 64),
          ([260] * 90, None, 8, 8, 16), ([260] * 90, None, 8, 8, 64), ([300, 277], None, 2, 2, 128), ([2100], None, 1, 1, 64),
          ([2500], None, 2, 1, 32), ([2085], None, 1, 1, 128), ([1, 2], [2777, 1500], 8, 2, 64), ([700], [5], 2, 2, 32)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("c", [1.0, 3.0])
@pytest.mark.parametrize("lq,lk,hq,hk,d", SHAPES)
def test_common_part_of_keys_and_values(lq, lk, hq, hk, d, c, dtype):
    from pymolecular_amd.segment_attention import segment_attention_backward, segment_attention_forward
    q, k, v, go, a, b = _case(lq, lk, hq, hk, d, dtype, seed=d)
    gen = torch.Generator().manual_seed(7)
    k, v = ((t.float() + c * torch.randn((1, hk, d), generator=gen).cuda()).to(dtype) for t in (k, v))
    q = (2 * q.float()).to(dtype)
    out, lse = segment_attention_forward(q, k, v, a, b)
    got = segment_attention_backward(go, q, k, v, out, lse, a, b)
    want = ref.segment_attention_grads_ref(_np(go), _np(q), _np(k), _np(v), a.cpu().numpy(), b.cpu().numpy())
    errs = [_rel(_np(x), y) for x, y in zip(got, want)]
    print([f"{e:.1e}" for e in errs], flush=True)
    tol = [1e-5 * (1 + c * c)] * 3 if dtype == F32 else [2 * 2.0 ** -9 * (1 + np.sqrt(1 + c * c)), 4 * 2.0 ** -9, 4 * 2.0 ** -9]
    assert all(e <= t for e, t in zip(errs, tol)), (errs, tol)
