"""Segment attention (egnn_attn_fwd / egnn_attn_bwd) against the float64 formulas of oracle.attention_ref.

Errors are normwise over a whole output, on inputs rounded to the dtype first.
  float32: products are exact to about one rounding, so a score of size s is off by about s 2^-23 and a probability by
      that, relatively; scores here stay below 40 and the sums average: bound 1e-5.
  bfloat16: one rounding of the output and one of the probabilities, each at most 2^-9 of a value: 2 x 2^-9 = 4e-3 for
      out.  The gradients also take the rounded out through delta = do . o and round p or ds: 4 x 2^-9 = 8e-3.
lse is held in fp32 in both: the scores' error (bfloat16 products are exact, their sums fp32), 1e-5 of its largest value.
"""
import numpy as np
import pytest
import torch

from oracle import attention_ref as ref

pytestmark = pytest.mark.gpu

TOL = {torch.float32: (1e-5, 1e-5), torch.bfloat16: (2 * 2.0 ** -9, 4 * 2.0 ** -9)}
F32, BF16 = torch.float32, torch.bfloat16


def _np(t):
    return t.detach().double().cpu().numpy()


def _off(lengths):
    return torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device="cuda")


def _rel(a, b):
    n = np.linalg.norm(b)
    return np.linalg.norm(a - b) / n if n else np.linalg.norm(a - b)


def _case(lq, lk, hq, hk, d, dtype, seed=0, packed=False, lead=0, tail=0):
    """q, k, v, go and the offsets; lead and tail rows lie outside every segment."""
    gen = torch.Generator().manual_seed(seed)
    nq, nk = sum(lq) + lead + tail, (sum(lq) if lk is None else sum(lk)) + lead + tail
    rand = lambda *s: torch.randn(s, generator=gen).to(dtype).cuda()  # noqa: E731
    if packed:
        w = rand(nq, hq + 2 * hk, d)
        q, k, v = w[:, :hq], w[:, hq:hq + hk], w[:, hq + hk:]
    else:
        q, k, v = rand(nq, hq, d), rand(nk, hk, d), rand(nk, hk, d)
    q_ptr = _off(lq) + lead
    kv_ptr = q_ptr if lk is None else _off(lk) + lead
    return q, k, v, rand(nq, hq, d), q_ptr, kv_ptr


def _both(q, k, v, go, q_ptr, kv_ptr, mask=None, scale=None):
    from pymolecular_amd.segment_attention import segment_attention_backward, segment_attention_forward
    out, lse = segment_attention_forward(q, k, v, q_ptr, kv_ptr, mask, scale)
    return out, lse, segment_attention_backward(go, q, k, v, out, lse, q_ptr, kv_ptr, mask, scale)


def _compare(q, k, v, go, q_ptr, kv_ptr, mask=None, scale=None):
    out, lse, grads = _both(q, k, v, go, q_ptr, kv_ptr, mask, scale)
    a = [_np(t) for t in (q, k, v)]
    m = None if mask is None else mask.cpu().numpy()
    ptrs = (q_ptr.cpu().numpy(), kv_ptr.cpu().numpy(), m, scale)
    o_ref, l_ref = ref.segment_attention_ref(*a, *ptrs)
    g_ref = ref.segment_attention_grads_ref(_np(go), *a, *ptrs)
    tol_o, tol_g = TOL[q.dtype]
    empty = np.isneginf(l_ref)
    assert np.array_equal(np.isneginf(_np(lse)), empty)
    errs = {"lse": np.abs(_np(lse) - l_ref)[~empty].max(initial=0) / max(1.0, np.abs(l_ref[~empty]).max(initial=0))}
    bounds = {"lse": 1e-5, "out": tol_o, "dq": tol_g, "dk": tol_g, "dv": tol_g}
    errs.update(out=_rel(_np(out), o_ref), **{n: _rel(_np(t), r) for n, t, r in zip(("dq", "dk", "dv"), grads, g_ref)})
    print({n: f"{e:.1e}" for n, e in errs.items()}, flush=True)
    bad = {n: e for n, e in errs.items() if not e <= bounds[n]}
    assert not bad, bad
    return out, lse, grads


SHAPES = [
    # lq, lk, heads, kv_heads, d
    ([9, 29, 17, 1, 2, 33], None, 4, 4, 32),            # molecules, a single atom, tiles of 16 and 32 crossed by one
    ([16, 32, 15, 31, 48], None, 8, 8, 16),             # tile edges
    ([1] * 70, [19] * 35 + [23] * 35, 4, 2, 32),        # one query a graph, more segments than one search round
    ([5, 0, 7], [0, 6, 40], 2, 1, 64),                  # no keys, no queries
    ([130, 64, 257], None, 2, 2, 64),                   # blocks of 64 rows, a tail row
    ([100, 301], [77, 129], 6, 2, 24),                  # cross attention, three heads share a key head, d not a power of 2
    ([67], None, 4, 1, 128),
    ([70, 3], None, 3, 3, 8),
    ([40, 90], None, 2, 2, 96),
    ([1], [2777], 8, 2, 64),                            # few rows, a long axis: split and joined
    ([900], [3], 4, 2, 32),                             # the same for dk and dv
    ([3, 2], [1500, 2500], 2, 2, 48),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lq,lk,hq,hk,d", SHAPES)
def test_matches_the_formulas(dtype, lq, lk, hq, hk, d):
    _compare(*_case(lq, lk, hq, hk, d, dtype, seed=d + len(lq)))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_scores_and_scales(dtype):
    q, k, v, go, a, b = _case([50, 21], None, 2, 2, 32, dtype, seed=3)
    for scale in (1.0, -0.25, 1e-3):                    # scores to about +-30, negated, nearly uniform
        _compare(q, k, v, go, a, b, scale=scale)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lq,lk", [([20, 9, 28, 150], None), ([4, 130], [200, 700]), ([1], [3000])])
def test_masked_keys(dtype, lq, lk):
    q, k, v, go, a, b = _case(lq, lk, 4, 2, 32, dtype, seed=5)
    gen = torch.Generator().manual_seed(1)
    mask = torch.rand(k.shape[0], generator=gen).cuda() < 0.6
    if len(lq) > 1:
        mask[int(b[0]):int(b[1])] = False               # a graph with no key left
    out, lse, (dq, dk, dv) = _compare(q, k, v, go, a, b, mask)
    assert torch.count_nonzero(dk[~mask]) == 0 and torch.count_nonzero(dv[~mask]) == 0
    if len(lq) > 1:
        assert torch.count_nonzero(out[:lq[0]]) == 0 and torch.count_nonzero(dq[:lq[0]]) == 0
    again = _both(q, k, v, go, a, b, mask.to(torch.uint8) * 7)
    assert torch.equal(out, again[0]) and all(torch.equal(x, y) for x, y in zip((dq, dk, dv), again[2]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_nothing_leaks(dtype, bad):
    # rows of another graph, masked keys, queries without keys and rows outside every graph hold NaN or infinities: the
    # other results are bit for bit those of clean inputs
    lq = [18, 25, 11, 100, 13]
    q, k, v, go, a, _ = _case(lq, None, 4, 2, 32, dtype, seed=9, lead=3, tail=5)
    mask = torch.ones(k.shape[0], dtype=torch.bool, device="cuda")
    s = [int(x) for x in a]
    mask[s[1] + 4] = mask[s[3] + 70] = False
    mask[s[4]:s[5]] = False                             # the last graph: no key left
    o0, _, g0 = _both(q, k, v, go, a, a, mask)
    q1, k1, v1, go1 = (t.clone() for t in (q, k, v, go))
    for t in (q1, k1, v1, go1):
        t[s[2]:s[3]] = bad                              # a whole graph
        t[:3] = bad
        t[-5:] = bad
        t[s[4]:s[5]] = bad
    for t in (k1, v1):
        t[s[1] + 4] = bad
        t[s[3] + 70] = bad
    o1, _, g1 = _both(q1, k1, v1, go1, a, a, mask)
    keep = torch.ones(q.shape[0], dtype=torch.bool, device="cuda")
    keep[s[2]:s[3]] = False
    for x, y in zip((o0, *g0), (o1, *g1)):
        assert torch.equal(x[keep], y[keep])
    for t in (o1, g1[0]):
        assert torch.count_nonzero(t[:3]) == 0 and torch.count_nonzero(t[-5:]) == 0 and torch.count_nonzero(t[s[4]:s[5]]) == 0
    assert not torch.isfinite(o1[s[2]:s[3]].float()).any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_key_has_no_score_gradient(dtype):
    # p = 1 whatever the score: dq and dk are 0 up to the rounding of do . v against do . o, dv is the sum of do
    q, k, v, go, a, b = _case([6, 40], [1, 1], 4, 2, 32, dtype, seed=2)
    out, _, (dq, dk, dv) = _both(q, k, v, go, a, b)
    size = _np(go).std() * _np(v).std() * _np(k).std()     # of one ds k: sqrt(32) scale = 1
    assert np.abs(_np(dq)).max() <= 32 * 2.0 ** -22 * size and np.abs(_np(dk)).max() <= 46 * 32 * 2.0 ** -22 * size
    assert _rel(_np(dv), ref.segment_attention_grads_ref(_np(go), _np(q), _np(k), _np(v), [0, 6, 46], [0, 1, 2])[2]) <= TOL[dtype][1]
    want = v[0].repeat_interleave(2, 0).expand(6, 4, 32)   # bfloat16: p rounds to 1; float32: p and the sum agree
    assert torch.equal(out[:6], want) if dtype == BF16 else (out[:6] - want).abs().max() <= 2.0 ** -22 * want.abs().max()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_views_and_widths(dtype):
    # parts of one projection are read where they lie, other strides are copied: the same results
    q, k, v, go, a, b = _case([30, 77], None, 4, 2, 32, dtype, seed=4, packed=True)
    want = _both(*(t.contiguous() for t in (q, k, v, go)), a, b)
    shifted = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)  # noqa: E731
    swapped = lambda t: t.transpose(0, 2).contiguous().transpose(0, 2)  # noqa: E731
    head_major = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    for f in (lambda t: t, shifted, swapped, head_major):
        got = _both(*(f(t) for t in (q, k, v, go)), a, b)
        assert torch.equal(got[0], want[0]) and all(torch.equal(x, y) for x, y in zip(got[2], want[2]))
    ones = torch.ones((), dtype=dtype, device="cuda").expand(q.shape)    # a sum's gradient: strides 0
    got, want = _both(q, k, v, ones, a, b), _both(q, k, v, ones.contiguous(), a, b)
    assert all(torch.equal(x, y) for x, y in zip(got[2], want[2]))
    _compare(*_case([20, 65], None, 2, 1, 19, dtype, seed=6))            # a width that the wrapper pads


def test_gradients_into_one_buffer():
    from pymolecular_amd.segment_attention import segment_attention_backward, segment_attention_forward
    q, k, v, go, a, _ = _case([30, 77], None, 4, 2, 32, BF16, seed=4, packed=True)
    out, lse = segment_attention_forward(q, k, v, a)
    want = segment_attention_backward(go, q, k, v, out, lse, a)
    buf = torch.full((q.shape[0], 8, 32), float("nan"), dtype=BF16, device="cuda")
    segment_attention_backward(go, q, k, v, out, lse, a, into=(buf[:, :4], buf[:, 4:6], buf[:, 6:]))
    assert torch.equal(buf, torch.cat(want, dim=1))


def test_gradient_against_differences():
    # d/dt of sum(go out(x + t u)) by central differences of the fp32 forward, u of unit-sized values: t = 2^-7 leaves
    # t^2 / 6 = 1e-5 of the third derivative, and rounding of 2^-24 sqrt(n) / t, 1e-6 of |grad| |u|
    from pymolecular_amd.segment_attention import segment_attention, segment_attention_forward
    q, k, v, go, a, b = _case([40, 19, 90], None, 4, 2, 32, F32, seed=8)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = segment_attention(*leaves, a)
    grads = torch.autograd.grad((out * go).sum(), leaves)
    gen = torch.Generator().manual_seed(0)
    for i in range(3):
        u = torch.randn(leaves[i].shape, generator=gen).cuda()
        u = u / u.norm() + grads[i] / grads[i].norm()   # not orthogonal to the gradient
        u = u * (u.numel() ** 0.5 / u.norm())

        def f(t):
            x = [y.detach() for y in leaves]
            x[i] = x[i] + t * u
            return (segment_attention_forward(*x, a)[0].double() * go.double()).sum()
        h = 2.0 ** -7
        num, ana = (f(h) - f(-h)) / (2 * h), (grads[i].double() * u.double()).sum()
        assert abs(num - ana) <= 2e-4 * grads[i].norm() * u.norm(), (i, num, ana)


def test_malformed_offsets_stay_in_bounds():
    # offsets past the rows are clamped, rows they leave out have no keys
    q, k, v, go, a, _ = _case([20, 30], None, 2, 2, 32, F32, seed=1)
    wild = torch.tensor([-5, 20, 4000], dtype=torch.int32, device="cuda")
    want = _both(q, k, v, go, a, a)
    got = _both(q, k, v, go, wild, wild)
    assert torch.equal(got[0], want[0]) and all(torch.equal(x, y) for x, y in zip(got[2], want[2]))
    part = torch.tensor([20], dtype=torch.int32, device="cuda")          # no segment at all
    out, lse, grads = _both(q, k, v, go, part, part)
    assert all(torch.count_nonzero(t) == 0 for t in (out, *grads)) and torch.isneginf(lse).all()


def test_no_rows():
    q, k, v, go, a, b = _case([0, 0], [3, 0], 2, 2, 32, BF16)
    out, lse, (dq, dk, dv) = _both(q, k, v, go, a, b)
    assert out.shape == (0, 2, 32) and lse.shape == (2, 0) and torch.count_nonzero(dk) == 0 and torch.count_nonzero(dv) == 0
    q, k, v, go, a, b = _case([4, 2], [0, 0], 2, 2, 32, BF16)
    out, _, (dq, dk, dv) = _both(q, k, v, go, a, b)
    assert torch.count_nonzero(out) == 0 and torch.count_nonzero(dq) == 0 and dk.shape == (0, 2, 32)


@pytest.mark.parametrize("lq,lk", [([18] * 40, None), ([600, 300], None), ([1], [5000])])
def test_same_bits_every_time_and_on_another_stream(lq, lk):
    args = _case(lq, lk, 8, 2, 64, BF16, seed=7)
    want = _both(*args)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = _both(*args)
    torch.cuda.current_stream().wait_stream(st)
    for x, y in zip((want[0], want[1], *want[2]), (got[0], got[1], *got[2])):
        assert torch.equal(x, y)


def test_under_a_graph():
    from pymolecular_amd.segment_attention import segment_attention_backward, segment_attention_forward
    q, k, v, go, a, b = _case([1, 3], [900, 1400], 4, 2, 32, BF16, seed=7)

    def step():
        out, lse = segment_attention_forward(q, k, v, a, b)
        return (out, *segment_attention_backward(go, q, k, v, out, lse, a, b))
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = step()
    for i in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)).to(BF16))
        want = [t.clone() for t in step()]
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(res, want))


def test_offsets_beyond_32_bits():
    # keys and values in rows of 192 values, 3.2e9 in all; a mask leaves a few keys, at both ends
    n = (1 << 24) + 3
    row = torch.zeros((n, 2, 96), dtype=BF16, device="cuda")
    keep = torch.tensor([0, 1, n // 2, n - 40, n - 2, n - 1], device="cuda")
    gen = torch.Generator().manual_seed(0)
    row[keep] = torch.randn((6, 2, 96), generator=gen).to(BF16).cuda()
    mask = torch.zeros(n, dtype=torch.bool, device="cuda")
    mask[keep] = True
    q = torch.randn((2, 1, 96), generator=gen).to(BF16).cuda()
    go = torch.randn((2, 1, 96), generator=gen).to(BF16).cuda()
    q_ptr = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    kv_ptr = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    out, _, (dq, dk, dv) = _both(q, row[:, :1], row[:, 1:], go, q_ptr, kv_ptr, mask)
    small = row[keep]
    args = [_np(t) for t in (q, small[:, :1], small[:, 1:])]
    o_ref, _ = ref.segment_attention_ref(*args, [0, 2], [0, 6])
    g_ref = ref.segment_attention_grads_ref(_np(go), *args, [0, 2], [0, 6])
    assert _rel(_np(out), o_ref) <= TOL[BF16][0]
    for x, r in zip((dq, dk[keep], dv[keep]), g_ref):
        assert _rel(_np(x), r) <= TOL[BF16][1]
    assert torch.count_nonzero(dk) <= 6 * 96 and torch.count_nonzero(dv) <= 6 * 96


def test_refusals():
    from pymolecular_amd.segment_attention import segment_attention, segment_attention_backward, segment_attention_forward
    q, k, v, go, a, _ = _case([20, 30], None, 4, 2, 32, F32)
    for args, err in [((q.half(), k.half(), v.half(), a), TypeError), ((q, k.to(BF16), v, a), TypeError),
                      ((q, k[:, :, :16], v, a), ValueError), ((q[:, :3], k, v, a), ValueError),
                      ((q, k, v, a.long()), ValueError), ((q, k, v, a, a[:2].clone()), ValueError),
                      ((q, k, v, a, None, torch.ones(49, dtype=torch.bool, device="cuda")), ValueError),
                      ((q, k, v, a, None, torch.ones(50, device="cuda")), ValueError),
                      ((q, k, v, a, None, None, 0.0), ValueError), ((q, k, v, a, None, None, float("nan")), ValueError),
                      ((q[:40], k, v, a), ValueError), ((q, k, v, a.cpu()), ValueError),
                      (tuple(torch.zeros(4, 1, 129, device="cuda") for _ in range(3)) + (a,), ValueError)]:
        with pytest.raises(err):
            segment_attention(*args)
    out, lse = segment_attention_forward(q, k, v, a)
    with pytest.raises(ValueError):
        segment_attention_backward(go[:, :2], q, k, v, out, lse, a)
    with pytest.raises(ValueError):
        segment_attention_backward(go, q, k, v, out, lse.t(), a)
    with pytest.raises(ValueError):
        segment_attention_backward(go, q, k, v, out, lse, a, into=(torch.empty_like(q), torch.empty_like(k), torch.empty_like(q)))


WIDE = [
    # 128-row tiles: enough of them, or a long segment that is split; each tile ends inside, at and past its last row
    ([260] * 60 + [256, 384, 1, 395], None, 8, 8, 64),
    ([2100], None, 1, 1, 64),
    ([2100], None, 2, 1, 32),
    ([2049, 5], None, 1, 1, 16),
    ([2085], None, 1, 1, 128),
    ([300, 2500], [2090, 4000], 2, 2, 32),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lq,lk,hq,hk,d", WIDE)
def test_wide_tiles(dtype, lq, lk, hq, hk, d):
    _compare(*_case(lq, lk, hq, hk, d, dtype, seed=len(lq)))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_wide_tiles_masked(dtype):
    q, k, v, go, a, b = _case([2100, 3], None, 2, 1, 32, dtype, seed=2, lead=2, tail=40)
    mask = torch.rand(k.shape[0], generator=torch.Generator().manual_seed(1)).cuda() < 0.5
    mask[100:900] = False                               # whole steps of masked keys
    mask[-43:] = False                                  # the second graph has none
    _compare(q, k, v, go, a, b, mask)


SHORT = [
    # segments of up to 32 rows among longer ones, on either axis
    ([20, 3, 150, 32, 33, 1, 0, 7] + [11] * 40, None, 4, 2, 32),
    ([8] * 30 + [40], [20] * 30 + [90], 4, 4, 32),
    ([12, 0, 9, 16, 17, 31], [9, 20, 0, 16, 90, 2], 4, 2, 64),
    ([5, 8, 9, 20], [32, 33, 7, 31], 8, 2, 16),         # 4 heads a key head: 20 to 80 rows
    ([2, 1, 30], [30, 30, 30], 3, 1, 40),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("lq,lk,hq,hk,d", SHORT)
def test_short_segments(dtype, masked, lq, lk, hq, hk, d):
    q, k, v, go, a, b = _case(lq, lk, hq, hk, d, dtype, seed=len(lq), lead=4, tail=50)
    mask = torch.rand(k.shape[0], generator=torch.Generator().manual_seed(3)).cuda() < 0.6 if masked else None
    _compare(q, k, v, go, a, b, mask)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_equal_offsets_in_two_tensors(dtype):
    # the same segments whether the axes share their offsets or not
    q, k, v, go, a, _ = _case([18, 25, 70, 32], None, 4, 2, 32, dtype, seed=1)
    want, got = _both(q, k, v, go, a, a), _both(q, k, v, go, a, a.clone())
    for x, y in zip((want[0], want[1], *want[2]), (got[0], got[1], *got[2])):
        assert torch.equal(x, y)


MANY_PARTS = [([1100, 1300], None, 4, 1, 64), ([2000], None, 2, 1, 32), ([700], [1500], 1, 1, 24)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lq,lk,hq,hk,d", MANY_PARTS)
def test_many_rows_in_many_parts(dtype, lq, lk, hq, hk, d):
    _compare(*_case(lq, lk, hq, hk, d, dtype, seed=len(lq)))
