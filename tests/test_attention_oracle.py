"""The float64 oracle's rows without keys: every output and gradient of them is 0."""
import numpy as np

from oracle import attention_ref as ref


def test_rows_without_keys_are_zero():
    r = np.random.Generator(np.random.PCG64(4))
    q, k, v, go = r.standard_normal((12, 4, 6)), r.standard_normal((15, 2, 6)), r.standard_normal((15, 2, 6)), r.standard_normal((12, 4, 6))
    mask = np.ones(15, dtype=bool)
    mask[7:10] = False                                    # the third segment's keys; the second has none; rows 11 and 13, 14 are outside
    seg = ([0, 5, 7, 9, 11], [0, 4, 4, 13, 13], mask)
    seg[1][2:4] = [7, 10]
    out, lse = ref.segment_attention_ref(q, k, v, *seg)
    dq, dk, dv = ref.segment_attention_grads_ref(go, q, k, v, *seg)
    none = [7, 8, 11]
    assert not out[none].any() and not dq[none].any() and np.isneginf(lse[:, none]).all()
    assert out[:7].all() and out[9:11].all() and np.isfinite(lse[:, [0, 1, 2, 3, 4, 5, 6, 9, 10]]).all()
    assert not dk[7:10].any() and not dv[7:10].any() and not dk[13:].any() and not dv[13:].any() and dv[:7].all()
