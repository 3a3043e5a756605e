"""Norm and rotation of heads against float64 on the CPU.

Bounds, in units of 2^-24 (a float32 rounding).  Forward: a sum of up to 128 squares in at most 23 additions one after the
other, whose square root takes half of it, a quotient and a root (2 + 1), two products, cos and sin (2 each: the series and
the argument's rounding) and a sum of two products: below 32 of the pair's length, plus half a step of the result.  Gradient
of the input, r (t - xh mean(t xh)): t carries the rotation and a product, xh the norm, their mean 24 additions more: below 64
of r (|t| + |xh| mean |t xh|), |t| that of the pair.  The weights' gradients sum n heads products: 2e-6 of their norm, as in
test_layer_norm_gpu.py, and half a step.
"""
import numpy as np
import pytest
import torch

from oracle.qk_ref import qk_norm_rotary_grads_ref, qk_norm_rotary_ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TYPES = [(F32, F32), (BF16, BF16), (BF16, F32)]


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _rand(seed, *shape, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _pair(x, rotary, il):
    """The length of the pair that each value belongs to."""
    out = np.abs(x)
    a, b = (np.arange(0, rotary, 2), np.arange(1, rotary, 2)) if il else (np.arange(rotary // 2), np.arange(rotary // 2, rotary))
    out[..., a] = out[..., b] = np.hypot(x[..., a], x[..., b])
    return out


def _close(y, want, size, units):
    err = np.abs(_np(y) - want)
    ok = err <= torch.finfo(y.dtype).eps / 2 * np.abs(want) * (1 + 1e-6) + units * 2.0 ** -24 * size
    assert ok.all(), (err.max(), (err / (size + 1e-30)).max() * 2 ** 24, np.argwhere(~ok)[:4])


def _inputs(n, hq, hk, d, rows, params, index, far, seed=0):
    q = _rand(seed, n, hq, d, dtype=rows) * (0.2 + _rand(seed + 1, 1, hq, 1, dtype=rows).abs())
    k = _rand(seed + 2, n, hk, d, dtype=rows) * 3
    if n > 2:
        q[1] = 0                              # a row of zeros: 0, and a gradient of 1 / sqrt(eps)
    gen = torch.Generator().manual_seed(seed + 3)
    hi = far if index == torch.int64 else min(far, 2 ** 31)
    pos = torch.randint(-hi, hi, (n,), generator=gen, dtype=torch.int64).to(index).cuda()
    return (q, k, (1 + 0.3 * _rand(seed + 4, d)).to(params), (1 + 0.3 * _rand(seed + 5, d)).to(params), pos,
            _rand(seed + 6, n, hq, d, dtype=rows), _rand(seed + 7, n, hk, d, dtype=rows))


def _compare(q, k, qw, kw, pos, gq, gk, base, rotary, il, eps=1e-6):
    from pymolecular_amd.qk_norm_rotary import qk_norm_rotary_backward, qk_norm_rotary_forward
    how = dict(base=base, rotary_dim=rotary, interleaved=il, eps=eps)
    outs = qk_norm_rotary_forward(q, k, qw, kw, pos, **how)
    grads = qk_norm_rotary_backward(gq, gk, q, k, qw, kw, pos, **how)
    again = qk_norm_rotary_backward(gq, gk, q, k, qw, kw, pos, **how)
    assert all(torch.equal(a, b) for a, b in zip(grads, again) if a is not None)
    p = None if pos is None else pos.cpu().numpy()
    for x, w, g, y, gx, gw in ((q, qw, gq, outs[0], grads[0], grads[2]), (k, kw, gk, outs[1], grads[1], grads[3])):
        assert y.dtype == gx.dtype == x.dtype and y.shape == gx.shape == x.shape
        xn, wn, gn = _np(x), _np(w), _np(g)
        want = qk_norm_rotary_ref(xn, wn, p, base, rotary, il, eps)
        _close(y, want, _pair(want, rotary, il), 32)
        wx, ww = qk_norm_rotary_grads_ref(gn, xn, wn, p, base, rotary, il, eps)
        r = 1 / np.sqrt((xn * xn).mean(-1, keepdims=True) + eps)
        big = np.abs(wn).max() if wn is not None else 1.0
        t, xh = _pair(gn, rotary, il) * big, xn * r
        _close(gx, wx, r * (t + np.abs(xh) * (t * np.abs(xh)).mean(-1, keepdims=True)), 64)
        if w is None:
            assert gw is None
        else:
            assert gw.dtype == w.dtype and gw.shape == w.shape
            err = np.linalg.norm(_np(gw) - ww)
            assert err <= (torch.finfo(gw.dtype).eps / 2 * (gw.dtype != F32) + 2e-6) * np.linalg.norm(ww) + 1e-30, err
    return outs, grads


CASES = [(1, 1, 1, 2, 2, False), (1, 1, 1, 2, 0, True), (64, 8, 2, 64, 64, False), (100, 4, 4, 32, 32, False),
         (333, 8, 8, 48, 24, True), (333, 8, 8, 48, 24, False), (41, 3, 1, 24, 12, False), (41, 2, 2, 24, 24, True),
         (77, 16, 4, 128, 128, False), (77, 2, 1, 128, 64, True), (50, 5, 5, 80, 80, False), (50, 4, 2, 96, 48, False),
         (19, 4, 2, 16, 8, False), (19, 7, 3, 16, 16, True), (30, 2, 2, 6, 6, False), (30, 2, 2, 34, 34, False),
         (30, 2, 2, 34, 2, True), (12, 2, 1, 126, 62, False), (12, 2, 1, 126, 126, False), (12, 2, 1, 126, 126, True),
         (9, 700, 30, 10, 4, False), (5000, 4, 1, 32, 32, False), (3001, 1, 1, 128, 128, True), (3, 4096, 1, 2, 2, False),
         (20000, 2, 2, 8, 8, False)]


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("rows,params", TYPES)
@pytest.mark.parametrize("n,hq,hk,d,rotary,il", CASES)
def test_values_and_gradients(n, hq, hk, d, rotary, il, rows, params, index):
    for far, base in ((500, 10000.0), (2 ** 32, 500000.0), (2 ** 20, 1.0)):
        q, k, qw, kw, pos, gq, gk = _inputs(n, hq, hk, d, rows, params, index, far, seed=d)
        _compare(q, k, qw, kw, pos, gq, gk, base, rotary, il)
        if far == 500:
            outs, grads = _compare(q, k, None, kw, pos, gq, gk, base, rotary, il, eps=1e-2)


@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("il", [False, True])
def test_strides_and_forms(rows, il):
    from pymolecular_amd.qk_norm_rotary import qk_norm_rotary, qk_norm_rotary_backward, qk_norm_rotary_forward
    q, k, qw, kw, pos, gq, gk = _inputs(90, 4, 2, 40, rows, rows, torch.int32, 1000)
    how = dict(rotary_dim=24, interleaved=il)
    want, grads = qk_norm_rotary_forward(q, k, qw, kw, pos, **how), qk_norm_rotary_backward(gq, gk, q, k, qw, kw, pos, **how)
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))  # noqa: E731
    wide = torch.full((90, 9, 43), float("nan"), dtype=rows, device="cuda")      # odd strides, misaligned heads
    wide[:, 1:5, 1:41], wide[:, 6:8, 3:43] = q, k
    a, b = wide[:, 1:5, 1:41], wide[:, 6:8, 3:43]
    assert same(qk_norm_rotary_forward(a, b, qw, kw, pos, **how), want)
    assert same(qk_norm_rotary_backward(gq, gk, a, b, qw, kw, pos, **how), grads)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, gq, gk)]
    assert same(qk_norm_rotary_forward(*heads_first[:2], qw, kw, pos, **how), want)
    assert same(qk_norm_rotary_backward(*heads_first[2:], *heads_first[:2], qw, kw, pos, **how), grads)
    apart = [t.permute(2, 0, 1).contiguous().permute(1, 2, 0) for t in (q, k, gq, gk)]   # a head's values apart: copied
    assert same(qk_norm_rotary_forward(*apart[:2], qw, kw, pos, **how), want)
    assert same(qk_norm_rotary_backward(*apart[2:], *apart[:2], qw, kw, pos, **how), grads)
    buf = torch.full((90, 8, 40), 7.0, dtype=rows, device="cuda")
    out = qk_norm_rotary_backward(gq, gk, q, k, qw, kw, pos, **how, into=(buf[:, :4], buf[:, 4:6]))
    assert same((buf[:, :4], buf[:, 4:6], *out[2:]), grads) and (buf[:, 6:] == 7).all()   # what lies between stays
    one = [t[:1].expand_as(t) for t in (q, k)]
    assert same(qk_norm_rotary(*one, qw, kw, pos, **how), qk_norm_rotary(*(t.contiguous() for t in one), qw, kw, pos, **how))
    wide_pos = torch.stack([pos, pos], 1)[:, 0]
    assert same(qk_norm_rotary_forward(q, k, qw, kw, wide_pos, **how), want)
    # no positions, no rows
    assert same(qk_norm_rotary(q, k, qw, kw), qk_norm_rotary(q, k, qw, kw, pos, rotary_dim=0))
    e = qk_norm_rotary_backward(gq[:0], gk[:0], q[:0], k[:0], qw, kw, pos[:0], **how)
    assert e[0].shape == (0, 4, 40) and not e[2].any() and not e[3].any()
    # a row with NaN or infinities spoils itself alone
    bad = q.clone()
    bad[7, 1], bad[8, 2, 3] = float("nan"), float("inf")
    keep = torch.ones((90, 4), dtype=torch.bool, device="cuda")
    keep[7, 1] = keep[8, 2] = False
    got = qk_norm_rotary_forward(bad, k, qw, kw, pos, **how)
    assert torch.equal(got[0][keep], want[0][keep]) and torch.equal(got[1], want[1])
    assert torch.equal(qk_norm_rotary_backward(gq, gk, bad, k, qw, kw, pos, **how)[0][keep], grads[0][keep])
    for args, err in (((q, k[:, :, :38]), ValueError), ((q[:89], k), ValueError), ((q, k.half()), TypeError),
                      ((q[:, :, :39], k[:, :, :39]), ValueError), ((q, k, qw[:39]), ValueError),
                      ((q, k, qw, kw, pos[:80]), ValueError), ((q, k, qw, kw, pos.float()), ValueError),
                      ((q, k, qw, kw, pos, 0.5), ValueError), ((q, k, qw, kw, pos, 1e4, 42), ValueError),
                      ((q, k, qw, kw, pos, 1e4, 7), ValueError), ((q, k, qw, kw, None, 1e4, 8), ValueError),
                      ((q, k, qw, kw, pos, 1e4, 8, False, -1.0), ValueError)):
        with pytest.raises(err):
            qk_norm_rotary(*args)
    with pytest.raises(ValueError, match="into"):
        qk_norm_rotary_backward(gq, gk, q, k, qw, kw, pos, **how, into=(buf[:1, :4].expand(90, 4, 40), buf[:, 4:6]))


@pytest.mark.parametrize("rows,params", TYPES + [(BF16, torch.float16), (F32, BF16)])
def test_autograd(rows, params):
    from pymolecular_amd.qk_norm_rotary import qk_norm_rotary
    q, k, qw, kw, pos, gq, gk = _inputs(120, 4, 2, 32, rows, params, torch.int64, 10000)
    leaves = [t.requires_grad_() for t in (q, k, qw, kw)]
    a, b = qk_norm_rotary(*leaves, pos)
    grads = torch.autograd.grad((a.float() * gq).sum() + (b.float() * gk).sum(), leaves)
    for x, w, g, gx, gw in ((q, qw, gq, grads[0], grads[2]), (k, kw, gk, grads[1], grads[3])):
        wx, ww = qk_norm_rotary_grads_ref(_np(g), _np(x), _np(w), pos.cpu().numpy())
        assert gx.dtype == x.dtype and gw.dtype == w.dtype
        for t, want in ((gx, wx), (gw, ww)):
            half = torch.finfo(t.dtype).eps / 2 if t.dtype != F32 else 0.0
            assert np.linalg.norm(_np(t) - want) <= (half + 4e-6) * np.linalg.norm(want)
    # differences of the float32 operator, over steps at which its rounding is 1e-3 of the change
    if rows == F32 and params == F32:
        u = _rand(9, 120, 4, 32) * q.detach().norm(dim=2, keepdim=True) / 32 ** 0.5
        u[1] = 0                              # (not at the row of zeros, where the norm bends within eps)
        h = 2.0 ** -8
        f = lambda t: float((qk_norm_rotary(t, k, qw, kw, pos)[0].double() * gq.double()).sum())  # noqa: E731
        with torch.no_grad():
            diff = (f(q + h * u) - f(q - h * u)) / (2 * h)
        size = float((grads[0].double() * u.double()).abs().sum())
        assert abs(diff - float((grads[0].double() * u.double()).sum())) <= 2e-3 * size
    g, = torch.autograd.grad((qk_norm_rotary(q, k, qw, kw, pos)[0] ** 2).sum() + (q ** 3).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(g.sum(), q)


@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("d,heads,kv", [(32, 4, 2), (32, 4, 4), (20, 4, 1), (128, 2, 1)])
def test_in_front_of_the_attention(rows, d, heads, kv):
    from pymolecular_amd.qk_norm_rotary import qk_norm_rotary, qk_norm_rotary_attention
    from pymolecular_amd.segment_attention import segment_attention
    lens = [12, 1, 0, 40, 87]
    seg = torch.tensor(np.cumsum([0] + lens), dtype=torch.int32, device="cuda")
    n = sum(lens)
    qkv = _rand(1, n, heads + 2 * kv, d, dtype=rows).requires_grad_()
    qw, kw = ((1 + 0.3 * _rand(s, d)).to(rows).requires_grad_() for s in (2, 3))
    pos = torch.cat([torch.arange(m) for m in lens]).cuda()
    mask = torch.rand(n, generator=torch.Generator().manual_seed(4)).cuda() < 0.8
    mask[13:53] = False                       # a graph whose keys are all left out
    go = _rand(5, n, heads, d, dtype=rows)
    out = qk_norm_rotary_attention(qkv, heads, seg, qw, kw, pos, mask, base=100.0, rotary_dim=d // 4 * 2)
    got = torch.autograd.grad((out * go).sum(), (qkv, qw, kw))
    q, k = qk_norm_rotary(qkv[:, :heads], qkv[:, heads:heads + kv], qw, kw, pos, 100.0, d // 4 * 2)
    plain = segment_attention(q, k, qkv[:, heads + kv:], seg, key_mask=mask)
    want = torch.autograd.grad((plain * go).sum(), (qkv, qw, kw))
    assert torch.equal(out, plain) and all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        assert torch.equal(qk_norm_rotary_attention(qkv, heads, seg, qw, kw, pos, mask, base=100.0, rotary_dim=d // 4 * 2), out)
        # only distances count: all positions moved by a number of their graph
        moved = pos + torch.repeat_interleave(torch.tensor([5, 9, 0, 1000, 70000]), torch.tensor(lens)).cuda()
        far = qk_norm_rotary_attention(qkv, heads, seg, qw, kw, moved, mask, base=100.0, rotary_dim=d // 4 * 2)
        # a rounding of q and k moves scores of up to 4 d^1/2 (weights up to 2) by half a step of that, twice
        step = torch.finfo(rows).eps / 2
        assert float((far - out).abs().max()) <= 64 * d ** 0.5 * step * float(qkv.abs().max())
    for bad in (0, heads + 2 * kv):
        with pytest.raises(ValueError):
            qk_norm_rotary_attention(qkv, bad, seg, qw, kw, pos)


def test_captured_and_on_another_stream():
    from pymolecular_amd.qk_norm_rotary import qk_norm_rotary_backward, qk_norm_rotary_forward
    q, k, qw, kw, pos, gq, gk = _inputs(500, 4, 2, 64, BF16, F32, torch.int32, 1000)
    run = lambda: (*qk_norm_rotary_forward(q, k, qw, kw, pos), *qk_norm_rotary_backward(gq, gk, q, k, qw, kw, pos))  # noqa: E731
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        first = run()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(first, run()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for seed in range(4):
        q.copy_(_rand(seed, 500, 4, 64))
        pos.add_(17)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, run()))


def test_offsets_past_32_bits():
    from pymolecular_amd.qk_norm_rotary import qk_norm_rotary_backward, qk_norm_rotary_forward
    n = 9_000_000
    x = _rand(1, 1000, 16, 32, dtype=BF16).repeat(n // 1000, 1, 1)
    pos = torch.arange(n, device="cuda") % 1000
    q, k = x[:, :8], x[:, 8:16]
    w = _rand(2, 32, dtype=BF16)
    outs = qk_norm_rotary_forward(q, k, w, w, pos)
    grads = qk_norm_rotary_backward(k, q, q, k, w, w, pos)
    few = qk_norm_rotary_forward(q[:1000], k[:1000], w, w, pos[:1000])
    gfew = qk_norm_rotary_backward(k[:1000], q[:1000], q[:1000], k[:1000], w, w, pos[:1000])
    for a, b in zip((*outs, *grads[:2]), (*few, *gfew[:2])):
        assert torch.equal(a[-1000:], b) and torch.equal(a[n // 2:n // 2 + 1000], b)
    for a, b in zip(grads[2:], gfew[2:]):
        # 9,000 times the sum: bf16 roundings of both, and 72,000,000 / 131,072 additions one after the other
        assert torch.allclose(a.float(), b.float() * (n // 1000), rtol=2 * 2.0 ** -8, atol=0.02 * float(b.float().abs().max()) * (n // 1000))
