"""Segment attention and layer norm under what records calls: a tracer, forward-mode differentiation, autograd.

Without a GPU the forward functions are replaced by ones that, like the library, work on addresses, where nothing sees
what they do.
"""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import pymolecular_amd.layer_norm as ln
import pymolecular_amd.segment_attention as sa


def _raw(f, *tensors):
    """f of the tensors' values, element by element, through their addresses."""
    out = torch.empty(tensors[0].shape)
    at = [(ctypes.c_float * out.numel()).from_address(t.data_ptr()) for t in (*tensors, out)]
    for i in range(out.numel()):
        at[-1][i] = f(*(a[i] for a in at[:-1]))
    return out


@pytest.fixture
def stand_in(monkeypatch):
    """out = 2 q + k + v, y = 3 x and the sum x + residual; the gradients are those of q k + v^2 / 2 and of x^2 / 2."""
    def attention(q, k, v, q_ptr, kv_ptr=None, key_mask=None, scale=None, need_lse=True):
        return _raw(lambda a, b, c: 2 * a + b + c, *(t.contiguous() for t in (q, k, v))), torch.zeros(q.shape[1], q.shape[0])

    def attention_backward(gout, q, k, v, out, lse, q_ptr, kv_ptr=None, key_mask=None, scale=None, into=None):
        g = [t.detach() * gout.detach() for t in (k, q, v)]
        for a, b in zip(into or (), g):
            a.copy_(b)
        return tuple(g)

    def norm(x, weight=None, bias=None, eps=1e-5, residual=None, need_stats=True):
        s = x if residual is None else _raw(lambda a, b: a + b, x, residual)
        return _raw(lambda a: 3 * a, x), s, torch.zeros(x.shape[0]), torch.ones(x.shape[0])

    def norm_backward(gy, s, weight, mean, rstd, gsum=None, need_weight=True, need_bias=True, **kw):
        return gy.detach() * s.detach(), torch.zeros(s.shape[-1]) if need_weight else None, torch.zeros(s.shape[-1]) if need_bias else None

    for m, name, f in ((sa, "segment_attention_forward", attention), (sa, "segment_attention_backward", attention_backward),
                       (ln, "layer_norm_forward", norm), (ln, "layer_norm_backward", norm_backward)):
        monkeypatch.setattr(m, name, f)


SEG = torch.tensor([0, 2, 5], dtype=torch.int32)
OPS = [
    # function of one tensor, its shape
    (lambda x: sa.segment_attention(x, x + 1, x - 1, SEG), (5, 2, 8)),
    (lambda x: sa.segment_attention_qkv(x, 2, SEG), (5, 6, 8)),
    (lambda x: ln.layer_norm(x), (4, 8)),
    (lambda x: ln.layer_norm(x, residual=x + 1)[0] + ln.layer_norm(x, residual=x + 1)[1], (4, 8)),
    (lambda x: ln.layer_norm(torch.ones(4, 8), weight=x[0]), (4, 8)),
]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("op,shape", OPS)
def test_traced_call_computes_again(stand_in, op, shape, grad):
    gen = torch.Generator().manual_seed(0)
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(op, torch.randn(shape, generator=gen), check_trace=False)
        for _ in range(2):
            x = torch.randn(shape, generator=gen)
            assert torch.equal(traced(x), op(x))


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("op,shape", OPS)
def test_a_tangent_is_refused(stand_in, op, shape, grad):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(0))
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        op(x)                                        # nothing is refused where no input has a tangent
        with pytest.raises(NotImplementedError):
            op(forward_ad.make_dual(x, torch.ones_like(x)))


SECOND = [
    # what meets the operator's output: nothing that depends on anything, and something that does
    lambda y: y.sum(), lambda y: (y * y).sum()]


def _second_order(op, x, f):
    # another path (x^3) keeps the first gradient differentiable: without the operator's part a second one would be wrong
    g, = torch.autograd.grad(f(op(x)) + (x ** 3).sum(), x, create_graph=True)
    plain, = torch.autograd.grad(f(op(x)) + (x ** 3).sum(), x)
    assert torch.equal(g, plain) and not plain.requires_grad
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(g.sum(), x)


@pytest.mark.parametrize("f", SECOND)
@pytest.mark.parametrize("op,shape", OPS)
def test_second_order_is_refused(stand_in, op, shape, f):
    _second_order(op, torch.randn(shape, generator=torch.Generator().manual_seed(0)).requires_grad_(), f)


def test_second_order_of_the_sum_alone(stand_in):
    x = torch.randn((4, 8), generator=torch.Generator().manual_seed(0)).requires_grad_()
    g, = torch.autograd.grad((ln.layer_norm(x, residual=2 * x)[1] ** 2).sum(), x, create_graph=True)
    assert torch.allclose(torch.autograd.grad(g.sum(), x)[0], torch.full_like(x, 18.0))


def _device_ops():
    gen = torch.Generator().manual_seed(1)
    seg = torch.tensor([0, 7, 40, 90], dtype=torch.int32, device="cuda")
    w, b, k, v = (torch.randn(s, generator=gen).cuda() for s in ((64,), (64,), (90, 2, 20), (90, 2, 20)))
    return [(lambda q: sa.segment_attention(q, k, v, seg), (90, 4, 20)),       # a width that the wrapper pads
            (lambda x: sa.segment_attention_qkv(x, 4, seg), (90, 8, 32)),
            (lambda x: ln.layer_norm(x, w, b), (90, 64)),
            (lambda x: sum(ln.layer_norm(x, w, b, residual=x * 0.5)), (90, 64)),
            (lambda x: ln.layer_norm(x[:, 1:], w[1:].contiguous()), (90, 64))]


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [False, True])
def test_traced_call_computes_again_on_the_device(grad):
    gen = torch.Generator().manual_seed(0)
    for op, shape in _device_ops():
        with torch.set_grad_enabled(grad):
            traced = torch.jit.trace(op, torch.randn(shape, generator=gen).cuda(), check_trace=False)
            for _ in range(2):
                x = torch.randn(shape, generator=gen).cuda()
                assert torch.equal(traced(x), op(x))


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [False, True])
def test_a_tangent_is_refused_on_the_device(grad):
    for op, shape in _device_ops():
        x = torch.randn(shape, generator=torch.Generator().manual_seed(0)).cuda()
        with torch.set_grad_enabled(grad), forward_ad.dual_level(), pytest.raises(NotImplementedError):
            op(forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.gpu
@pytest.mark.parametrize("f", SECOND)
def test_second_order_is_refused_on_the_device(f):
    for op, shape in _device_ops():
        _second_order(op, torch.randn(shape, generator=torch.Generator().manual_seed(0)).cuda().requires_grad_(), f)
