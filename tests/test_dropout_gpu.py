"""Dropout, and layer norm of residual + dropout, against float64 on the CPU.

Bounds.  A value that stays is x up: up is rounded to float32 (2^-24 of it at most; exact for p = 0 and 1/2), the product
(2^-24), the sum with the residual (2^-24 of the sum), and the result to its dtype (half a step, eps / 2).  fp32 norms and
gradients are held to 2e-6 normwise and bf16 ones to 2 x 2^-9, as in test_layer_norm_gpu.py.  Gradients are those of the sum
before it is rounded: exactly beside float32 parameters, else to 2^-17 of it, which adds up to 2^-16 |mean| / std beside a
rounding of 2^-8.
"""
import numpy as np
import pytest
import torch

from oracle import attention_ref as ref
from oracle.dropout_ref import dropout_grad_ref, dropout_ref, keep_ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
SEED, OFFSET = -(2 ** 61) + 12345, 2 ** 33 - 2


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _rng(seed=SEED, offset=OFFSET):
    return torch.tensor([seed, offset], dtype=torch.int64, device="cuda")


def _rand(seed, *shape, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _close(y, want, scaled):
    """y against want = residual + scaled (module docstring)."""
    half = torch.finfo(y.dtype).eps / 2
    err = np.abs(_np(y) - want)
    ok = err <= (half + 2.0 ** -23) * np.abs(want) + 2.0 ** -22 * np.abs(scaled)
    assert ok.all(), (err.max(), np.argwhere(~ok)[:4])


SHAPES = [(1, 1), (1, 8), (77, 128), (300, 5), (41, 259), (3, 10007), (2049, 16), (2, 8193), (129, 1024), (5, 40000)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,c", SHAPES)
def test_values(n, c, dtype):
    from pymolecular_amd.dropout import dropout_backward, dropout_forward
    x, r = _rand(1, n, c, dtype=dtype), _rand(2, n, c, dtype=dtype)
    for p in (0.0, 0.1, 0.5, 0.9999, 1.0):
        want = dropout_ref(_np(x), p, SEED, OFFSET + 3)
        y = dropout_forward(x, p, _rng(), site=3)
        assert y.dtype == dtype
        _close(y, want, want)
        assert np.array_equal(_np(y) == 0, (want == 0) | (_np(x) == 0))         # the mask, value by value
        assert torch.equal(dropout_backward(x, p, _rng(), site=3), y)
        _close(dropout_forward(x, p, _rng(), r, site=3), want + _np(r), want)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_shapes_and_dtypes(dtype):
    from pymolecular_amd.dropout import dropout_forward
    rng = _rng()
    x = _rand(3, 50, 99, dtype=dtype)
    want = dropout_forward(x, 0.25, rng, x)
    wide = torch.full((50, 107), float("nan"), dtype=dtype, device="cuda")
    wide[:, 5:104] = x
    assert torch.equal(dropout_forward(wide[:, 5:104], 0.25, rng, wide[:, 5:104]), want)     # odd strides, misaligned rows
    assert torch.equal(dropout_forward(x.t().contiguous().t(), 0.25, rng, x), want)            # columns apart
    assert torch.equal(dropout_forward(x.view(5, 10, 99), 0.25, rng, x.view(5, 10, 99)), want.view(5, 10, 99))
    one = x[:1].expand(50, 99)                                                               # rows all the same one
    assert torch.equal(dropout_forward(one, 0.25, rng), dropout_forward(one.contiguous(), 0.25, rng))
    assert dropout_forward(x[:0], 0.25, rng).shape == (0, 99)
    assert torch.equal(dropout_forward(x[0], 0.25, rng), dropout_forward(x, 0.25, rng)[0])     # one row
    other = BF16 if dtype == F32 else F32
    y = dropout_forward(x, 0.25, rng, x.to(other))
    assert y.dtype == F32 and torch.equal(y, dropout_forward(x.float(), 0.25, rng, x.to(other).float()))
    with pytest.raises(TypeError):
        dropout_forward(x.half(), 0.25, rng)
    for bad in (x[:, :98], x[:49]):
        with pytest.raises(ValueError):
            dropout_forward(x, 0.25, rng, bad)


def test_what_is_dropped_may_be_anything():
    from pymolecular_amd.dropout import dropout
    from pymolecular_amd.layer_norm import layer_norm_dropout_forward
    from pymolecular_amd.dropout import Dropout
    keep, _ = keep_ref(64, 40, 0.5, SEED, OFFSET)
    x = _rand(4, 64, 40)
    bad = torch.where(torch.from_numpy(keep).cuda(), x, torch.tensor([float("nan"), float("inf")], device="cuda").repeat(64, 20))
    assert torch.equal(dropout(bad, 0.5, _rng(), x), dropout(x, 0.5, _rng(), x))
    for a, b in zip(*(layer_norm_dropout_forward(t, x, Dropout(0.5, _rng())) for t in (bad, x))):
        assert torch.equal(a, b)


def test_autograd():
    from pymolecular_amd.dropout import dropout
    x, r, gy = _rand(5, 30, 41).requires_grad_(), _rand(6, 30, 41, dtype=BF16).requires_grad_(), _rand(7, 30, 41)
    rng = _rng()
    gx, gr = torch.autograd.grad((dropout(x, 0.3, rng, r, site=9) * gy).sum(), (x, r))
    want = dropout_grad_ref(_np(gy), 0.3, SEED, OFFSET + 9)
    _close(gx, want, want)
    assert gr.dtype == BF16 and torch.equal(gr, gy.to(BF16))
    # by differences: the operator is linear, so any step will do but for the rounding of the sums
    u = _rand(8, 30, 41)
    f = lambda t: (dropout(t, 0.3, rng, site=9).double() * gy.double()).sum()  # noqa: E731
    with torch.no_grad():
        assert abs(float((f(x + u) - f(x - u)) / 2 - (gx.double() * u.double()).sum())) < 30 * 41 * 2.0 ** -20
    # again differentiable: the gradient of the gradient is the mask once more
    y = dropout(x, 0.3, rng)
    g, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    h, = torch.autograd.grad((g * gy).sum(), x)
    want = 2 * dropout_ref(dropout_ref(_np(gy), 0.3, SEED, OFFSET), 0.3, SEED, OFFSET)
    _close(h, want, 2 * want)
    # a generator that was advanced in between is refused
    y = dropout(x, 0.3, rng)
    rng[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


NORMS = [(1, 1), (77, 128), (300, 5), (41, 259), (64, 8), (9, 1000), (3, 4099), (2, 12289), (300, 1536), (65601, 42),
         (33, 24), (5, 700)]


@pytest.mark.parametrize("dtype,params", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("n,c", NORMS)
def test_norm(n, c, dtype, params):
    from pymolecular_amd.dropout import Dropout, dropout_forward
    from pymolecular_amd.layer_norm import layer_norm_dropout_backward, layer_norm_dropout_forward
    x, gy, gs = (_rand(i, n, c, dtype=dtype) for i in (1, 2, 3))
    r = (_rand(4, n, c) + 0.5 * _rand(5, n, 1)).to(dtype)
    w, b = (1 + 0.2 * _rand(6, c)).to(params), _rand(7, c).to(params)
    drop = Dropout(0.1, _rng(), 5)
    y, s, mean, rstd = layer_norm_dropout_forward(x, r, drop, w, b)
    assert torch.equal(s, dropout_forward(x, 0.1, drop.rng, r, site=5))
    y_ref, s_ref = ref.layer_norm_ref(dropout_ref(_np(x), 0.1, SEED, OFFSET + 5), _np(w), _np(b), 1e-5, _np(r))
    tol = 2e-6 if dtype == F32 else 2 * 2.0 ** -9
    rel = lambda a, t: np.linalg.norm(_np(a) - t) / max(np.linalg.norm(t), 1e-30)  # noqa: E731
    if c > 1:                                 # (a row of one value has y = bias, and no gradient: rounding divided by eps)
        assert rel(y, y_ref) <= tol
    for gsum in (None, gs):
        grads = layer_norm_dropout_backward(gy, s, drop, w, mean, rstd, gsum)
        gr, gw, gb = ref.layer_norm_grads_ref(_np(gy), s_ref, _np(w), 1e-5, _np(gsum))
        gx = dropout_grad_ref(gr, 0.1, SEED, OFFSET + 5)
        assert [t.dtype for t in grads] == [dtype, dtype, params, params]
        errs = [rel(a, t) for a, t in zip(grads, (gx, gr, gw, gb))] if c > 1 else [0.0]
        print([f"{e:.1e}" for e in errs], flush=True)
        assert max(errs) <= tol and max(errs[2:], default=0.0) <= (2e-6 if params == F32 else tol)
        assert np.array_equal(_np(grads[0]) == 0, (gx == 0) | (_np(grads[1]) == 0))


@pytest.mark.parametrize("params", [BF16, F32])
@pytest.mark.parametrize("n,c", [(3000, 40), (3000, 259), (300, 4099)])
def test_gradients_of_the_unrounded_sum(n, c, params):
    # rows whose mean is four times their deviation: the stored sum's rounding would be 1e-2 of them
    from pymolecular_amd.dropout import Dropout
    from pymolecular_amd.layer_norm import layer_norm_dropout_backward, layer_norm_dropout_forward
    x, gy = (_rand(i, n, c, dtype=BF16) for i in (1, 2))
    r = (_rand(3, n, c) + 4 * _rand(4, n, 1).sign()).to(BF16)
    w, b = (1 + 0.2 * _rand(5, c)).to(params), _rand(6, c).to(params)
    drop = Dropout(0.25, _rng(), 1)
    y, s, mean, rstd = layer_norm_dropout_forward(x, r, drop, w, b)
    s_ref = dropout_ref(_np(x), 0.25, SEED, OFFSET + 1, _np(r))
    gr, gw, gb = ref.layer_norm_grads_ref(_np(gy), s_ref, _np(w))
    got = layer_norm_dropout_backward(gy, s, drop, w, mean, rstd)
    rel = lambda a, t: np.linalg.norm(_np(a) - t) / np.linalg.norm(t)  # noqa: E731
    # one rounding of the result, at most half a step; the statistics' 2^-24 |mean| / std, the sum's 2^-17 |mean| / std
    half = 2.0 ** -8 if params == BF16 else 0.0
    assert rel(got[1], gr) <= 2.0 ** -8 + 2.0 ** -14
    assert rel(got[2], gw) <= half + (2.0 ** -14 if params == BF16 else 4e-6) and rel(got[3], gb) <= half + 2e-6
    # rows of one value (no deviation): the gradient is 0 but for the gradient of the sum
    one = torch.full((n, 1), 1.37, dtype=BF16, device="cuda")
    y, s, mean, rstd = layer_norm_dropout_forward(x[:, :1].contiguous(), one, drop, w[:1], b[:1])
    got = layer_norm_dropout_backward(gy[:, :1].contiguous(), s, drop, w[:1], mean, rstd)
    assert float(got[1].float().abs().max()) == 0.0 == float(got[2].float().abs().max())
    # a bias alone, and what another call returned
    y, s, mean, rstd = layer_norm_dropout_forward(x, r, drop, None, b)
    assert torch.equal(layer_norm_dropout_backward(gy, s, drop, None, mean, rstd, bias_dtype=params)[1],
                       layer_norm_dropout_backward(gy, s, drop, None, mean, rstd, need_bias=False)[1])
    with pytest.raises(ValueError, match="rstd"):
        layer_norm_dropout_backward(gy, s, drop, None, mean, (rstd[0], rstd[1][:1]))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_autograd_and_forms(dtype):
    from pymolecular_amd.dropout import Dropout, dropout
    from pymolecular_amd.layer_norm import layer_norm, layer_norm_dropout
    rng = _rng()
    n, c = 40, 60
    leaves = [_rand(1, n, c, dtype=dtype), _rand(2, n, c), 1 + 0.1 * _rand(3, c), _rand(4, c)]
    gy, gs = _rand(5, n, c), _rand(6, n, c)

    def grads(f):
        t = [a.clone().requires_grad_() for a in leaves]
        y, s = f(*t)
        return (y, s, *torch.autograd.grad((y * gy).sum() + (s * gs).sum(), t))

    got = grads(lambda x, r, w, b: layer_norm_dropout(x, r, Dropout(0.25, rng, 2), w, b))
    want = grads(lambda x, r, w, b: layer_norm(dropout(x.float(), 0.25, rng, site=2), w, b, residual=r))
    tol = 2e-6 if dtype == F32 else 2 * 2.0 ** -8
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and float((a - b).detach().double().norm()) <= tol * float(b.detach().double().norm())
    # the sum alone, the norm alone, nothing recorded
    x, r = (t.clone().requires_grad_() for t in leaves[:2])
    gx, gr = torch.autograd.grad((layer_norm_dropout(x, r, Dropout(0.25, rng))[1] * gs).sum(), (x, r))
    assert torch.equal(gr, gs) and torch.equal(gx, dropout(gs, 0.25, rng).to(dtype))
    with torch.no_grad():
        y, s = layer_norm_dropout(x, r, Dropout(0.25, rng, 2), leaves[2], leaves[3])
    assert torch.equal(y, got[0]) and torch.equal(s, got[1])
    # rows that are parts of wider ones
    wide = torch.zeros((n, c + 5), dtype=dtype, device="cuda")
    wide[:, 3:3 + c] = leaves[0]
    y2, s2 = layer_norm_dropout(wide[:, 3:3 + c], r.detach(), Dropout(0.25, rng, 2), leaves[2], leaves[3])
    assert torch.equal(y2, y) and torch.equal(s2, s)
    g, = torch.autograd.grad(layer_norm_dropout(x, r, Dropout(0.25, rng))[0].sum() + (x ** 3).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(g.sum(), x)
    y, _ = layer_norm_dropout(x, r, Dropout(0.25, rng))
    rng[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_captured_graph_draws_anew():
    from pymolecular_amd.dropout import Dropout, dropout_backward, dropout_forward
    from pymolecular_amd.layer_norm import layer_norm_dropout_backward, layer_norm_dropout_forward
    x, r, gy, w, b = _rand(1, 100, 128), _rand(2, 100, 128), _rand(3, 100, 128), _rand(4, 128), _rand(5, 128)
    state = _rng()

    def step(rng):
        rng[1] += 4
        d = Dropout(0.1, rng, 1)
        y, s, mean, rstd = layer_norm_dropout_forward(x, r, d, w, b)
        return [dropout_forward(x, 0.1, rng, r), dropout_backward(gy, 0.1, rng), y, s,
                *layer_norm_dropout_backward(gy, s, d, w, mean, rstd)]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(_rng())
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(state)
    eager = _rng()
    last = None
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        want = step(eager)
        assert all(torch.equal(a, t) for a, t in zip(outs, want)) and torch.equal(state, eager)
        assert last is None or not torch.equal(outs[0], last)
        last = outs[0].clone()


def test_another_stream():
    from pymolecular_amd.dropout import dropout_forward
    x = _rand(1, 4000, 128)
    want = dropout_forward(x, 0.1, _rng())
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        z = x * 0 + x
        y = dropout_forward(z, 0.1, _rng())
    stream.synchronize()
    assert torch.equal(y, want)


def test_more_rows_than_one_launch():
    # 2^20 workgroups a launch: one row of 8192 values each here, four rows of 512 in the norm
    from pymolecular_amd.dropout import Dropout, dropout_forward
    from pymolecular_amd.layer_norm import layer_norm_dropout_forward
    n = (1 << 20) + 3
    y = dropout_forward(torch.ones((1, 8192), dtype=BF16, device="cuda").expand(n, 8192), 0.5, _rng())
    for lo in (0, n - 7):
        assert np.array_equal(_np(y[lo:lo + 7]), dropout_ref(np.ones((7, 8192)), 0.5, SEED, OFFSET, row0=lo))
    del y
    n = (4 << 20) + 5
    s = layer_norm_dropout_forward(torch.ones((n, 512), dtype=BF16, device="cuda"), torch.zeros((n, 512), dtype=BF16, device="cuda"),
                                   Dropout(0.5, _rng()), need_stats=False)[1]
    assert np.array_equal(_np(s[-9:]), dropout_ref(np.ones((9, 512)), 0.5, SEED, OFFSET, row0=n - 9))
