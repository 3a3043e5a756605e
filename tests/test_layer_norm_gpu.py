"""Layer norm (egnn_norm_fwd / egnn_norm_bwd) against the float64 formulas of oracle.attention_ref.

Errors are normwise over a whole output.  float32: a handful of roundings a value and sums of at most a few hundred
terms in a row: bound 2e-6 (the weight's gradient, summed over the rows: the same).  bfloat16: one rounding of the
output, 2^-9 at most; the gradients of x and the weight are made from the stored sum, whose rounding weighs |s| / std s
(1 to 2 in these rows) in (s - mean) / std: 2 x 2^-9, and 4 x 2^-9 for those two.
"""
import numpy as np
import pytest
import torch

from oracle import attention_ref as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TOL = {F32: 2e-6, BF16: 2 * 2.0 ** -9}
TOL_S = {F32: 2e-6, BF16: 4 * 2.0 ** -9}


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _rel(a, b):
    return np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-300)


def _inputs(n, c, dtype, residual, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    x = (rand(n, c) * (0.5 + rand(n, 1).abs()) + 0.3 * rand(n, 1)).to(dtype).cuda()
    r = rand(n, c).to(dtype).cuda() if residual else None
    w, b = (1 + 0.2 * rand(c)).to(dtype).cuda(), rand(c).to(dtype).cuda()
    return x, r, w, b, rand(n, c).to(dtype).cuda(), (rand(n, c).to(dtype).cuda() if residual else None)


def _compare(x, r, w, b, gy, gs, eps=1e-5):
    from pymolecular_amd.layer_norm import layer_norm_backward, layer_norm_forward
    y, s, mean, rstd = layer_norm_forward(x, w, b, eps, r)
    got = layer_norm_backward(gy, s, w, mean, rstd, gs)
    y_ref, s_ref = ref.layer_norm_ref(_np(x), _np(w), _np(b), eps, _np(r))
    g_ref = ref.layer_norm_grads_ref(_np(gy), s_ref, _np(w), eps, _np(gs))
    errs = {n: _rel(_np(t), a) for n, t, a in zip(("y", "s", "gx", "gw", "gb"), (y, s, *got), (y_ref, s_ref, *g_ref))}
    print({n: f"{e:.1e}" for n, e in errs.items()}, flush=True)
    bad = {n: e for n, e in errs.items() if not e <= (TOL_S if n in ("gx", "gw") else TOL)[x.dtype]}
    assert not bad, bad


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("n,c", [(1, 128), (77, 128), (1000, 64), (333, 256), (50, 16), (41, 259), (9, 1000), (130, 8),
                                 (17, 5), (3, 4096), (5, 5000), (70, 515), (12, 1027), (6, 12289)])
def test_matches_the_formulas(n, c, dtype, residual):
    _compare(*_inputs(n, c, dtype, residual, seed=c))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_rows(dtype):
    _compare(*_inputs(60001, 128, dtype, True, seed=1))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("c", [128, 100, 2200])
def test_strided_rows_and_no_parameters(dtype, c):
    from pymolecular_amd.layer_norm import layer_norm_backward, layer_norm_forward
    x, r, w, b, gy, gs = _inputs(57, c, dtype, True, seed=3)
    wide = lambda t, off: torch.zeros((57, 2 * c + 11), dtype=dtype, device="cuda")[:, off:off + c].copy_(t)  # noqa: E731
    for off in (0, 8, 3):
        _compare(*(wide(t, off) for t in (x, r)), w, b, *(wide(t, off) for t in (gy, gs)))
    y, s, mean, rstd = layer_norm_forward(x)
    gx, gw, gb = layer_norm_backward(gy, s, None, mean, rstd, need_weight=False, need_bias=False)
    assert gw is None and gb is None and s is x
    assert _rel(_np(y), ref.layer_norm_ref(_np(x))[0]) <= TOL[dtype]
    assert _rel(_np(gx), ref.layer_norm_grads_ref(_np(gy), _np(x))[0]) <= TOL[dtype]
    ones = torch.ones((), dtype=dtype, device="cuda").expand(57, c)     # a sum's gradient: stride 0
    assert all(torch.equal(p, q) for p, q in zip(layer_norm_backward(ones, s, w, mean, rstd),
                                                 layer_norm_backward(ones.contiguous(), s, w, mean, rstd)))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_column_and_constant_rows(dtype):
    from pymolecular_amd.layer_norm import layer_norm, layer_norm_backward, layer_norm_forward
    b = torch.randn(1, generator=torch.Generator().manual_seed(0)).to(dtype).cuda()
    x = torch.randn(40, 1, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    assert torch.equal(layer_norm(x, None, b), b.expand(40, 1))          # s = mean s
    c = torch.full((5, 128), 3.0, dtype=dtype, device="cuda")            # variance 0: rstd = eps^-1/2
    y, s, mean, rstd = layer_norm_forward(c, eps=1e-5)
    assert torch.count_nonzero(y) == 0 and torch.allclose(rstd, torch.full_like(rstd, 1e-5 ** -0.5), rtol=1e-6)
    gx, _, _ = layer_norm_backward(torch.ones_like(c), s, None, mean, rstd)
    assert gx.abs().max() <= 128 * 2.0 ** -23 * 1e-5 ** -0.5


def test_bad_rows_stay_rows():
    # NaN or an infinity in a row changes that row's results and the weight's gradient, and no other row
    from pymolecular_amd.layer_norm import layer_norm_backward, layer_norm_forward
    for c in (128, 99, 3000):
        x, _, w, b, gy, _ = _inputs(37, c, F32, False, seed=2)
        y0, s0, m0, r0 = layer_norm_forward(x, w, b)
        g0 = layer_norm_backward(gy, s0, w, m0, r0)[0]
        x1 = x.clone()
        x1[5, 3], x1[20, 0] = float("nan"), float("inf")
        y1, s1, m1, r1 = layer_norm_forward(x1, w, b)
        g1 = layer_norm_backward(gy, s1, w, m1, r1)[0]
        keep = [i for i in range(37) if i not in (5, 20)]
        assert torch.equal(y0[keep], y1[keep]) and torch.equal(g0[keep], g1[keep])
        assert torch.isnan(y1[5]).all() and torch.isnan(y1[20]).any()


def test_autograd_and_sum_only():
    from pymolecular_amd.layer_norm import layer_norm
    x, r, w, b, gy, gs = _inputs(50, 96, F32, True, seed=4)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
    y, s = layer_norm(leaves[0], leaves[1], leaves[2], residual=leaves[3])
    got = torch.autograd.grad((y * gy).sum() + (s * gs).sum(), leaves, retain_graph=True)
    want = ref.layer_norm_grads_ref(_np(gy), _np(x) + _np(r), _np(w), 1e-5, _np(gs))
    for t, a in zip(got, (*want, want[0])):
        assert _rel(_np(t), a) <= TOL[F32]
    only = torch.autograd.grad((s * gs).sum(), [leaves[0], leaves[3]])
    assert torch.equal(only[0], gs) and torch.equal(only[1], gs)
    z = layer_norm(x.view(5, 10, 96), w, b)                             # leading axes are rows
    assert z.shape == (5, 10, 96) and torch.equal(z.view(50, 96), layer_norm(x, w, b))


def test_gradient_against_differences():
    # central differences of the fp32 forward, step 2^-5: t^2 / 6 of the third derivative and rounding, below 2e-3
    from pymolecular_amd.layer_norm import layer_norm_backward, layer_norm_forward
    x, _, w, b, gy, _ = _inputs(30, 131, F32, False, seed=6)
    _, s, mean, rstd = layer_norm_forward(x, w, b)
    gx, gw, gb = layer_norm_backward(gy, s, w, mean, rstd)
    h = 2.0 ** -5
    for i, g in ((0, gx), (1, gw), (2, gb)):
        u = g / g.norm() + torch.randn(g.shape, generator=torch.Generator().manual_seed(i)).cuda() / g.numel() ** 0.5

        def f(t):
            a = [x, w, b]
            a[i] = a[i] + t * u
            return (layer_norm_forward(*a)[0].double() * gy.double()).sum()
        num, ana = (f(h) - f(-h)) / (2 * h), (g.double() * u.double()).sum()
        assert abs(num - ana) <= 2e-3 * g.norm() * u.norm(), i


def test_no_rows_and_same_bits():
    from pymolecular_amd.layer_norm import layer_norm_backward, layer_norm_forward
    x, r, w, b, gy, gs = _inputs(20000, 128, BF16, True, seed=8)
    y, s, mean, rstd = layer_norm_forward(x, w, b, residual=r)
    one = layer_norm_backward(gy, s, w, mean, rstd, gs)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        two = layer_norm_backward(gy, s, w, mean, rstd, gs)
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    y, s, mean, rstd = layer_norm_forward(x[:0], w, b)
    gx, gw, gb = layer_norm_backward(gy[:0], s, w, mean, rstd)
    assert y.shape == (0, 128) and torch.count_nonzero(gw) == 0 and torch.count_nonzero(gb) == 0


def test_under_a_graph():
    from pymolecular_amd.layer_norm import layer_norm_backward, layer_norm_forward
    x, r, w, b, gy, gs = _inputs(3000, 256, BF16, True, seed=8)

    def step():
        y, s, mean, rstd = layer_norm_forward(x, w, b, residual=r)
        return (y, s, *layer_norm_backward(gy, s, w, mean, rstd, gs))
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = step()
    for i in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(i)).to(BF16))
        want = [t.clone() for t in step()]
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(res, want))


def test_refusals():
    from pymolecular_amd.layer_norm import layer_norm, layer_norm_backward, layer_norm_forward
    x, r, w, b, gy, _ = _inputs(10, 32, F32, True)
    for args, kw, err in [((x.half(),), {}, TypeError), ((x, w[:31]), {}, ValueError), ((x, w, b.cpu()), {}, ValueError),
                          ((x, w, b), dict(residual=r[:9]), ValueError), ((x, w, b), dict(eps=-1.0), ValueError),
                          ((x[:, :0],), {}, ValueError)]:
        with pytest.raises(err):
            layer_norm(*args, **kw)
    _, s, mean, rstd = layer_norm_forward(x, w, b)
    with pytest.raises(ValueError):
        layer_norm_backward(gy[:5], s, w, mean, rstd)
    with pytest.raises(ValueError):
        layer_norm_backward(gy, s, w, mean[:5], rstd)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,c", [(70001, 42), (66003, 91), (65601, 165), (65541, 331), (65536, 160)])
def test_many_rows_of_odd_widths(n, c, dtype):
    # a row's last piece overlaps the one before; many rows take three pieces a lane
    _compare(*_inputs(n, c, dtype, n % 2 == 0, seed=c))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("c", [1, 3, 4, 7, 8, 9, 15, 31, 33, 255, 257, 511, 513])
def test_widths_around_a_piece(c, dtype):
    _compare(*_inputs(37, c, dtype, True, seed=c))
