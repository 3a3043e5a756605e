"""Table rows, dropout, and normed and turned heads in forms that their own tests do not reach: under a tracer and
forward-mode differentiation, two calls at once on two streams, tables whose partial sums need more than one launch's
workgroups."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _rand(seed, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _ops():
    """(function of one float tensor, its shape)"""
    from pymolecular_amd.dropout import Dropout, dropout
    from pymolecular_amd.embedding import embedding
    from pymolecular_amd.layer_norm import layer_norm_dropout
    from pymolecular_amd.qk_norm_rotary import qk_norm_rotary, qk_norm_rotary_attention
    rng = torch.tensor([3, 4], device="cuda")
    tokens, pos = torch.arange(90, device="cuda") % 7, torch.arange(90, device="cuda")
    seg = torch.tensor([0, 7, 40, 90], dtype=torch.int32, device="cuda")
    w, hw = _rand(1, 64), _rand(2, 32)
    return [(lambda x: embedding(tokens, x, 2.0), (7, 64)),
            (lambda x: embedding(tokens, x[:, 1:], 2.0, dtype=BF16).float(), (7, 64)),
            (lambda x: dropout(x, 0.2, rng), (90, 64)),
            (lambda x: dropout(x[:, 1:], 0.2, rng, x[:, :-1]), (90, 64)),
            (lambda x: sum(layer_norm_dropout(x, x * 0.5, Dropout(0.2, rng, 1), w, w)), (90, 64)),
            (lambda x: sum(layer_norm_dropout(x[:, 1:], x[:, 1:], Dropout(0.2, rng, 1))), (90, 64)),
            (lambda x: sum(qk_norm_rotary(x[:, :4], x[:, 2:6], hw, hw, pos)), (90, 6, 32)),
            (lambda x: qk_norm_rotary_attention(x, 4, seg, hw, hw, pos), (90, 8, 32)),
            (lambda x: qk_norm_rotary_attention(x, 4, seg, positions=pos, rotary_dim=10), (90, 6, 20))]


@pytest.mark.parametrize("grad", [False, True])
def test_traced_call_computes_again(grad):
    for op, shape in _ops():
        with torch.set_grad_enabled(grad):
            traced = torch.jit.trace(op, _rand(5, *shape), check_trace=False)
            for seed in (6, 7):
                x = _rand(seed, *shape)
                assert torch.equal(traced(x), op(x))


@pytest.mark.parametrize("grad", [False, True])
def test_a_tangent_is_refused(grad):
    for op, shape in _ops():
        x = _rand(5, *shape)
        with torch.set_grad_enabled(grad), forward_ad.dual_level(), pytest.raises(NotImplementedError):
            op(forward_ad.make_dual(x, torch.ones_like(x)))


def test_second_derivatives():
    for i, (op, shape) in enumerate(_ops()):
        x = _rand(5, *shape).requires_grad_()
        g, = torch.autograd.grad((op(x) ** 2).sum() + (x ** 3).sum(), x, create_graph=True)
        plain, = torch.autograd.grad((op(x) ** 2).sum() + (x ** 3).sum(), x)
        assert torch.equal(g, plain)
        if i in (2, 3):                       # the dropout is linear in x: its gradient can be differentiated again
            # f = sum (A x)^2 + x^3 for a linear A: grad of sum(grad f) is 2 A^T A 1 + 6 x
            ones = torch.ones_like(x).requires_grad_()
            want, = torch.autograd.grad((op(ones) ** 2).sum(), ones)
            h, = torch.autograd.grad(g.sum(), x)
            assert torch.allclose(h, want + 6 * x, rtol=1e-5, atol=1e-5)
        else:
            with pytest.raises(RuntimeError, match="no second derivative"):
                torch.autograd.grad(g.sum(), x)


def test_two_calls_at_once():
    from pymolecular_amd.embedding import embedding_backward
    from pymolecular_amd.qk_norm_rotary import qk_norm_rotary_backward
    t = [(torch.arange(60000, device="cuda") * m) % v for m, v in ((7, 100), (11, 30000), (13, 90), (17, 20000))]
    g = _rand(1, 60000, 64, dtype=BF16)
    q = _rand(2, 4000, 4, 64, dtype=BF16)
    pos, w = torch.arange(4000, device="cuda"), _rand(3, 64, dtype=BF16)
    calls = [lambda i=i: embedding_backward(g, t[i], 30000) for i in range(4)] + [
        lambda s=s: qk_norm_rotary_backward(q, q, q, q, w, w, pos + s)[2] for s in range(2)]
    want = [f() for f in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None] * len(calls)
    for _ in range(3):
        for i, f in enumerate(calls):
            with torch.cuda.stream(streams[i % 2]):
                got[i] = f()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_wide_partial_tables():
    # partial tables of 2^28 values: more pieces than one launch has workgroups
    from pymolecular_amd.embedding import embedding_backward
    n, v, c = 4100, 1000, 1 << 18
    tokens = torch.cat([torch.arange(n - 50, device="cuda") % v, torch.full((50,), 7, device="cuda")])
    row = torch.randint(-3, 4, (1, c), generator=torch.Generator().manual_seed(0)).to(BF16).cuda()
    gw = embedding_backward(row.expand(n, c), tokens, v, 2.0, 5)
    count = torch.bincount(tokens, minlength=v).float()
    count[5] = 0
    for a in range(0, v, 100):
        assert torch.equal(gw[a:a + 100].float(), (2 * count[a:a + 100, None] * row.float()).to(BF16).float())
