"""Heads that an attention leaves out, masked keys and rows outside every segment, may hold NaN and infinities: with their
norm and rotation in front of it, they reach neither the weights' gradients nor those of other rows, and get 0."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
ODD = [float("nan"), float("inf"), -float("inf"), 3e38]


def _rand(seed, *shape, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("rows,params", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("d,heads,kv,il", [(32, 4, 2, False), (48, 4, 4, True), (10, 2, 1, False), (128, 3, 1, True), (2, 4, 4, False)])
def test_heads_without_a_gradient(rows, params, d, heads, kv, il):
    from pymolecular_amd.qk_norm_rotary import qk_norm_rotary_backward
    n = 700
    q, gq = (_rand(s, n, heads, d, dtype=rows) for s in (1, 2))
    k, gk = (_rand(s, n, kv, d, dtype=rows) for s in (3, 4))
    w = (1 + 0.3 * _rand(5, 2, d)).to(params)
    pos = torch.arange(n, device="cuda")
    gen = torch.Generator().manual_seed(6)
    zq, zk = (torch.rand((n, h), generator=gen).cuda() < 0.3 for h in (heads, kv))
    gq[zq], gk[zk] = 0, 0
    want = qk_norm_rotary_backward(gq, gk, q, k, w[0], w[1], pos, interleaved=il)
    bad = []
    for t, z in ((q, zq), (k, zk)):
        odd = torch.tensor(ODD, device="cuda").to(rows)[torch.randint(0, 4, t.shape, generator=gen).cuda()]
        few = odd.where(torch.rand(t.shape, generator=gen).cuda() < 0.5, t)          # a part of the head, or all of it
        few = few.where((torch.arange(n, device="cuda") % 2 == 0)[:, None, None], odd)
        bad.append(few.where(z[..., None], t))
    got = qk_norm_rotary_backward(gq, gk, *bad, w[0], w[1], pos, interleaved=il)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert not got[0][zq].any() and not got[1][zk].any()
    # one value of the gradient is enough to take part
    gq[zq.nonzero()[0][0], zq.nonzero()[0][1], d - 1] = 1
    assert qk_norm_rotary_backward(gq, gk, torch.full_like(q, float("nan")), k, w[0], w[1], pos, interleaved=il)[2].isnan().all()


@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("d,heads,kv", [(32, 4, 2), (20, 4, 1), (128, 2, 2)])
def test_left_out_by_the_attention(rows, d, heads, kv):
    from pymolecular_amd.qk_norm_rotary import qk_norm_rotary_attention
    n = 400
    seg = torch.tensor([7, 40, 40, 220, 360], dtype=torch.int32, device="cuda")      # rows in front of and behind all segments
    mask = torch.rand(n, generator=torch.Generator().manual_seed(4)).cuda() < 0.7
    mask[40:60] = False
    outside = torch.ones(n, dtype=torch.bool, device="cuda")
    outside[7:360] = False
    qkv, go = _rand(1, n, heads + 2 * kv, d, dtype=rows), _rand(2, n, heads, d, dtype=rows)
    bad = qkv.clone()
    bad[outside] = torch.tensor(ODD, device="cuda").to(rows).repeat(n)[:d]
    bad[~mask & ~outside, heads:] = float("nan")

    def run(x):
        t = [x.clone().requires_grad_(), *((1 + 0.3 * _rand(s, d)).to(rows).requires_grad_() for s in (5, 6))]
        out = qk_norm_rotary_attention(t[0], heads, seg, t[1], t[2], torch.arange(n, device="cuda"), mask)
        return (out, *torch.autograd.grad((out * go).sum(), t))

    got, want = run(bad), run(qkv)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert not got[0][outside].any() and not got[1][outside].any() and not got[1][~mask, heads:].any()


@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("d", [32, 10])
def test_heads_of_zeros_without_eps(rows, d):
    # 0 / 0 in the forward, as the formula has it; without a gradient (a batch padded with zeros) such heads get 0
    from pymolecular_amd.qk_norm_rotary import qk_norm_rotary_backward
    q, gq, w, pos = _rand(1, 90, 4, d, dtype=rows), _rand(2, 90, 4, d, dtype=rows), _rand(3, 2, d, dtype=rows), torch.arange(90, device="cuda")
    gq[70:], gq[:, 3] = 0, 0
    want = qk_norm_rotary_backward(gq, gq, q, q, w[0], w[1], pos, eps=0.0)
    q[70:], q[::2, 3] = 0, 0
    got = qk_norm_rotary_backward(gq, gq, q, q, w[0], w[1], pos, eps=0.0)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and not got[0][70:].any()
