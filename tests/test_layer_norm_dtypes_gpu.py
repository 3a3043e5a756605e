"""Layer norm where the parameters or the residual have another dtype than the rows.

Bounds.  What leaves in float32 from exact inputs is held to float32's, 2e-6 normwise, as in test_layer_norm_gpu.py: gw and
gb beside bfloat16 rows without a residual (the rows are exact), everything of a float32 sum.  A bfloat16 value is the
rounding of one that is right to float32: |y - y_ref| <= 2^-8 |y_ref| + 2^-18 (values of about 1 to 8 before the rounding).
A parameter rounded to bfloat16 first would miss the latter by up to twice as much, and the former by 1e-3.
"""
import numpy as np
import pytest
import torch

from oracle import attention_ref as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _rel(a, b):
    return np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-300)


def _rounded(y, want):
    return (np.abs(_np(y) - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -18).all()


def _inputs(n, c, seed):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    x = (rand(n, c) * (0.5 + rand(n, 1).abs()) + 0.3 * rand(n, 1)).to(BF16).cuda()
    return x, (1 + 0.2 * rand(c)).cuda(), rand(c).cuda(), rand(n, c).to(BF16).cuda(), rand(n, c).cuda()


@pytest.mark.parametrize("n,c", [(77, 128), (300, 5), (41, 259), (64, 8), (9, 1000), (3, 4099), (20001, 64), (65601, 42)])
def test_float32_parameters_beside_bfloat16_rows(n, c):
    from pymolecular_amd.layer_norm import layer_norm, layer_norm_backward, layer_norm_forward
    x, w, b, gy, _ = _inputs(n, c, c)
    y, s, mean, rstd = layer_norm_forward(x, w, b)
    gx, gw, gb = layer_norm_backward(gy, s, w, mean, rstd)
    assert y.dtype == gx.dtype == BF16 and gw.dtype == gb.dtype == F32
    g_ref = ref.layer_norm_grads_ref(_np(gy), _np(x), _np(w))
    errs = [_rel(_np(t), g) for t, g in zip((gw, gb), g_ref[1:])]
    print(errs, flush=True)
    assert _rounded(y, ref.layer_norm_ref(_np(x), _np(w), _np(b))[0])
    assert max(errs) <= 2e-6 and _rel(_np(gx), g_ref[0]) <= 2 * 2.0 ** -9
    # by autograd the parameters' gradients are those, and a strided input's the same
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad((layer_norm(*leaves) * gy).sum(), leaves)
    assert all(torch.equal(p, q) for p, q in zip(got, (gx, gw, gb)))
    wide = torch.zeros((n, c + 3), dtype=BF16, device="cuda")
    wide[:, 3:] = x
    assert torch.equal(layer_norm(wide[:, 3:], w, b), y)


@pytest.mark.parametrize("c", [128, 99, 4099])
def test_each_parameter_in_a_dtype_of_its_own(c):
    from pymolecular_amd.layer_norm import layer_norm
    x, w, b, gy, _ = _inputs(50, c, c + 1)
    for wt, bt in ((w, b.to(BF16)), (w.to(BF16), b), (None, b), (w, None), (w.half(), b.half())):
        leaves = [t.detach().clone().requires_grad_() for t in (x, wt, bt) if t is not None]
        it = iter(leaves[1:])
        y = layer_norm(leaves[0], *(None if t is None else next(it) for t in (wt, bt)))
        assert _rounded(y, ref.layer_norm_ref(_np(x), _np(wt), _np(bt))[0])
        got = torch.autograd.grad((y * gy).sum(), leaves)
        want = ref.layer_norm_grads_ref(_np(gy), _np(x), _np(wt))
        for t, leaf, g in zip(got, leaves, [want[0]] + [a for a, p in zip(want[1:], (wt, bt)) if p is not None]):
            tol = {F32: 2e-6, torch.float16: 2.0 ** -11, BF16: 2.0 ** -8}[leaf.dtype]
            assert t.dtype == leaf.dtype and _rel(_np(t), g) <= tol
    # float32 rows: bfloat16 parameters lose nothing, their gradients are rounded once
    y = layer_norm(x.float(), w.to(BF16), b)
    assert y.dtype == F32 and _rel(_np(y), ref.layer_norm_ref(_np(x), _np(w.to(BF16)), _np(b))[0]) <= 2e-6


@pytest.mark.parametrize("c", [128, 99, 4099])
def test_a_residual_of_another_dtype(c):
    # the sum, and what is made from it, in the dtype of x + residual; gradients in those of the inputs
    from pymolecular_amd.layer_norm import layer_norm
    x, w, b, gy, r = _inputs(50, c, c + 2)
    gs = torch.randn((50, c), generator=torch.Generator().manual_seed(3)).cuda()
    for u, v in ((x, r), (r, x)):
        leaves = [t.detach().clone().requires_grad_() for t in (u, v, w, b)]
        y, s = layer_norm(leaves[0], leaves[2], leaves[3], residual=leaves[1])
        assert y.dtype == s.dtype == F32 and torch.equal(s, u + v)
        assert _rel(_np(y), ref.layer_norm_ref(_np(s), _np(w), _np(b))[0]) <= 2e-6
        got = torch.autograd.grad((y * gy).sum() + (s * gs).sum(), leaves)
        gx, gw, gb = ref.layer_norm_grads_ref(_np(gy), _np(s), _np(w), 1e-5, _np(gs))
        for t, leaf, g in zip(got, leaves, (gx, gx, gw, gb)):
            assert t.dtype == leaf.dtype and _rel(_np(t), g) <= (2e-6 if t.dtype == F32 else 2.0 ** -8)
    with pytest.raises(TypeError):
        layer_norm(x, w, b, residual=r.double())


def test_a_network_of_float32_parameters_on_bfloat16_nodes():
    # the norms of such a network get the gradients that float32 parameters accumulate
    from pymolecular_amd import graphs
    from pymolecular_amd.models.EGNN import EGNNGlobal
    torch.manual_seed(0)
    g = graphs.molecule_batch(5, seed=1, feat_seed=2)
    net = EGNNGlobal(5, 128, 1, n_layers=1, heads=4, kv_heads=2).cuda()
    edges = tuple(torch.from_numpy(a.astype(np.int64)).cuda() for a in (g.rows(), g.col))
    seg = torch.tensor([int(o) for o in g.info["graph_offsets"]], dtype=torch.int32, device="cuda")
    out, h, _ = net(torch.from_numpy(g.node_feat).to(BF16).cuda(), torch.from_numpy(g.coord).float().cuda(), edges, None, seg)
    assert out.dtype == h.dtype == BF16
    h.backward(torch.randn(h.shape, generator=torch.Generator().manual_seed(1)).to(BF16).cuda())
    for norm in (net.gcl_norm_0, net.att_norm_0):
        for p in (norm.weight, norm.bias):
            assert p.grad.dtype == F32 and not torch.equal(p.grad, p.grad.to(BF16).float())
