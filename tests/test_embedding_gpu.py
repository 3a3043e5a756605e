"""Table rows by token and the table's gradient against float64 on the CPU.

Bounds.  The forward rounds scale to float32, the product, and the result to its dtype: 2^-24 each of the value and half a
step.  Gradients of small integers with a scale of 2 are exact in float32 in any order, and are compared for equality.  Others
carry at most one rounding an addition: the longest chain of additions is one of at most 600 (eight rows at a time over the
span of a group of lanes, up to 512 groups of a workgroup, 64 partial sums in turn), so 602 x 2^-24 of the sum of the absolute
values, and half a step of the result.
"""
import numpy as np
import pytest
import torch

from oracle.embedding_ref import embedding_grad_ref, embedding_ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TYPES = [(F32, F32), (BF16, BF16), (BF16, F32)]


def _np(t):
    return t.detach().double().cpu().numpy()


def _tokens(n, v, skew, seed, dtype=torch.int64, outside=True):
    gen = torch.Generator().manual_seed(seed)
    t = (torch.rand(n, generator=gen, dtype=torch.float64) ** skew * v).long().clamp(max=v - 1)
    if outside and n > 8:   # tokens outside the table, near and far
        far = [-1, v, -(1 << 31), (1 << 31) - 1] + ([1 << 32, (1 << 40) + 3, -(1 << 62)] if dtype == torch.int64 else [])
        at = torch.randperm(n, generator=gen)[:len(far)]
        t[at] = torch.tensor(far)
    return t.to(dtype).cuda()


def _rand(seed, *shape, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _ints(seed, *shape, dtype=F32):
    return torch.randint(-3, 4, shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("rows,table", TYPES)
@pytest.mark.parametrize("n,v,c", [(1, 1, 1), (77, 119, 128), (300, 7, 5), (41, 1000, 259), (9, 3, 10007), (2049, 50, 16),
                                   (5000, 20, 3)])
def test_forward(n, v, c, rows, table, index):
    from pymolecular_amd.embedding import embedding, embedding_forward
    t, w = _tokens(n, v, 1.0, n, index), _rand(1, v, c, dtype=table)
    for scale in (1.0, c ** 0.5):
        out = embedding_forward(t, w, scale, dtype=rows)
        want = embedding_ref(t.cpu().numpy(), _np(w), scale)
        assert out.dtype == rows and (np.abs(_np(out) - want) <= (torch.finfo(rows).eps / 2 + 2.0 ** -22) * np.abs(want)).all()
    wide = torch.full((v, c + 3), float("nan"), dtype=table, device="cuda")
    wide[:, 2:2 + c] = w
    assert torch.equal(embedding(t, wide[:, 2:2 + c], c ** 0.5, dtype=rows), out)        # rows of a wider table, misaligned
    assert torch.equal(embedding(t.view(1, n), w, c ** 0.5, dtype=rows), out.view(1, n, c))
    assert torch.equal(embedding(torch.stack([t, t], 1)[:, 0], w, c ** 0.5, dtype=rows), out)


# the form with one workgroup a range of the table (up to 4,096 tokens), chunks with partial tables, sorted
SIZES = [(1, 1, 1), (1, 50000, 20), (64, 3, 5), (1000, 119, 128), (4096, 1025, 8), (3, 2000, 2500), (4000, 100000, 16),
         (4097, 2, 7), (6145, 119, 128), (20000, 119, 128), (65601, 119, 42), (70000, 1000, 24), (30001, 5, 259), (50000, 1, 64),
         (6144, 9000, 33), (9000, 4500, 130), (12345, 1023, 64), (40961, 50021, 40), (70001, 131072, 16), (30000, 20000, 1),
         (9001, 8191, 1030), (20000, 1100000, 4)]


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("rows,table", TYPES)
@pytest.mark.parametrize("n,v,c", SIZES)
def test_gradient(n, v, c, rows, table, index):
    from pymolecular_amd.embedding import embedding_backward
    for skew, padding in ((1.0, None), (4.0, 0), (40.0, v - 1)):
        t = _tokens(n, v, skew, n + c, index)
        tn = t.cpu().numpy()
        g = _ints(2, n, c, dtype=rows)
        got = embedding_backward(g, t, v, 2.0, padding, dtype=table)
        assert got.dtype == table and got.shape == (v, c)
        want = torch.from_numpy(embedding_grad_ref(_np(g), tn, v, 2.0, padding)).to(table)
        bad = (got.cpu() != want).any(1).nonzero().flatten()
        assert not len(bad), (skew, bad[:8].tolist(), len(bad))
    g = _rand(3, n, c, dtype=rows)
    got = embedding_backward(g, t, v, 0.3, padding, dtype=table)
    want, size = embedding_grad_ref(_np(g), tn, v, 0.3, padding), embedding_grad_ref(np.abs(_np(g)), tn, v, 0.3, padding)
    err = np.abs(_np(got) - want)
    assert (err <= torch.finfo(table).eps / 2 * np.abs(want) + 602 * 2.0 ** -24 * size).all()
    assert torch.equal(got, embedding_backward(g, t, v, 0.3, padding, dtype=table))       # the same bits every time


@pytest.mark.parametrize("n,v", [(3000, 100), (30000, 100), (30000, 30000)])
def test_orders_and_what_no_token_may_reach(n, v):
    from pymolecular_amd.embedding import embedding_backward
    c = 40
    g = _ints(4, n, c)
    cases = {"one token": torch.full((n,), v // 2), "sorted": torch.arange(n) * v // n, "reversed": v - 1 - torch.arange(n) * v // n,
             "the last row": torch.full((n,), v - 1), "none inside": torch.full((n,), -5), "all behind": torch.full((n,), v),
             "alternating": torch.arange(n) % 2 * (v - 1)}
    for name, t in cases.items():
        t = t.cuda()
        got = embedding_backward(g, t, v, 2.0)
        assert np.array_equal(_np(got), embedding_grad_ref(_np(g), t.cpu().numpy(), v, 2.0)), name
    # NaN and infinities of padding and of tokens outside the table reach nothing
    t = _tokens(n, v, 2.0, 5)
    out = (t < 0) | (t >= v) | (t == 7)
    bad = torch.where(out[:, None], torch.tensor([float("nan"), float("inf")], device="cuda").repeat(n, c // 2), g)
    assert torch.equal(embedding_backward(bad, t, v, 2.0, 7), embedding_backward(g, t, v, 2.0, 7))
    # rows apart, all the same one, misaligned
    wide = torch.full((n, c + 5), float("nan"), device="cuda")
    wide[:, 3:3 + c] = g
    want = embedding_backward(g, t, v, 2.0)
    assert torch.equal(embedding_backward(wide[:, 3:3 + c], t, v, 2.0), want)
    one = g[:1].expand(n, c)
    assert torch.equal(embedding_backward(one, t, v, 2.0), embedding_backward(one.contiguous(), t, v, 2.0))
    assert torch.equal(embedding_backward(g.view(n // 10, 10, c), t.view(n // 10, 10), v, 2.0), want)
    assert not embedding_backward(g[:0], t[:0], v).any()


def test_autograd_and_dtypes():
    from pymolecular_amd.embedding import embedding
    t = _tokens(500, 30, 2.0, 1)
    go = _rand(2, 500, 24)
    for table, rows in ((F32, None), (F32, BF16), (BF16, None), (BF16, F32), (torch.float16, F32), (torch.float16, BF16)):
        w = _rand(3, 30, 24, dtype=table).requires_grad_()
        out = embedding(t, w, 1.5, 2, dtype=rows)
        assert out.dtype == (table if rows is None else rows)
        want = embedding_ref(t.cpu().numpy(), _np(w), 1.5)
        assert (np.abs(_np(out) - want) <= (torch.finfo(out.dtype).eps / 2 + 2.0 ** -22) * np.abs(want)).all()
        g, = torch.autograd.grad((out * go.to(out.dtype)).sum(), w)
        assert g.dtype == table
        gr = _np(go.to(out.dtype))
        want, size = (embedding_grad_ref(a, t.cpu().numpy(), 30, 1.5, 2) for a in (gr, np.abs(gr)))
        # (float16 tables: float32 sums, rounded once more)
        assert (np.abs(_np(g) - want) <= torch.finfo(table).eps / 2 * 1.01 * np.abs(want) + 602 * 2.0 ** -24 * size).all()
    w = _rand(3, 30, 24).requires_grad_()
    u = _rand(4, 30, 24)
    g, = torch.autograd.grad((embedding(t, w, 1.5) * go).sum(), w)
    with torch.no_grad():                    # linear: differences of any step
        f = lambda x: float((embedding(t, x, 1.5).double() * go.double()).sum())  # noqa: E731
        assert abs((f(w + u) - f(w - u)) / 2 - float((g.double() * u.double()).sum())) < 500 * 24 * 2.0 ** -18
    g, = torch.autograd.grad((embedding(t, w) ** 2).sum() + (w ** 3).sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(g.sum(), w)
    for bad in (lambda: embedding(t.float(), w), lambda: embedding(t, w.double(), dtype=torch.float64)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: embedding(t, w.cpu()), lambda: embedding(t, w, float("nan")), lambda: embedding(t, w, 1.0, 30)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("n,v", [(1000, 100), (20000, 100), (20000, 50000)])
def test_captured_and_on_another_stream(n, v):
    from pymolecular_amd.embedding import embedding_backward, embedding_forward
    t, g, w = _tokens(n, v, 2.0, 1), _rand(2, n, 72), _rand(3, v, 72)
    run = lambda: (embedding_forward(t, w, 2.0), embedding_backward(g, t, v, 0.5, 3))  # noqa: E731
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
        t.copy_(_tokens(n, v, 1.0 + seed, seed))
        g.copy_(_rand(seed + 10, n, 72))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, run()))


def test_long_tables_and_many_tokens():
    # offsets past 2^32 bytes and 2^31 values in the table, its gradient, the rows and theirs
    from pymolecular_amd.embedding import embedding_backward, embedding_forward
    v, c = 2_200_000, 1024
    w = torch.zeros((v, c), dtype=BF16, device="cuda")
    t = torch.tensor([v - 1, 5, v - 2, v - 1, 2_100_000], device="cuda")
    w[t] = _ints(1, 5, c, dtype=BF16)
    w[v - 1] = 2.0
    out = embedding_forward(t, w, 2.0)
    assert torch.equal(out, (2 * w[t].float()).to(BF16))
    gw = embedding_backward(out, t, v, 2.0)
    assert torch.equal(gw[v - 1], torch.full((c,), 16.0, dtype=BF16, device="cuda")) and torch.equal(gw[v - 2], 2 * out[2])
    assert int((gw != 0).any(1).sum()) <= 4
    del w, out, gw
    n = 2_200_000
    tokens = torch.arange(n, device="cuda") % 50
    rows = embedding_forward(tokens, _ints(2, 50, c, dtype=BF16), 1.0)
    assert torch.equal(rows[-50:], rows[:50]) and torch.equal(rows[n // 2: n // 2 + 50], rows[:50])
    for vocab in (50, 60000):                  # partial tables, sorted
        gw = embedding_backward(rows, tokens, vocab, 2.0 ** -4, dtype=BF16)
        assert torch.equal(gw[:50].float(), (rows[:50].float() * (n // 50) * 2.0 ** -4).to(BF16).float()) and not gw[50:].any()
