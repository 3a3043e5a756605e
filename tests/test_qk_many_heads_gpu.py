"""Norm and rotation of thousands of narrow query heads beside one key head, in tiles of hundreds of rows: every head is by
itself, so the rows of a large call are those of a call on a few of them, bit for bit.  The rows of the large call are all the
same one in memory; the positions tell them apart."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("hq,hk", [(4095, 1), (1, 2931)])
def test_rows_of_large_tiles(hq, hk):
    from pymolecular_amd.qk_norm_rotary import qk_norm_rotary_backward, qk_norm_rotary_forward
    n, d = (1 << 19) + 5, 2
    gen = torch.Generator().manual_seed(hq)
    q, k, gq, gk = (torch.randn((1, h, d), generator=gen).to(BF16).cuda().expand(n, h, d) for h in (hq, hk, hq, hk))
    w = torch.randn((2, d), generator=gen).to(BF16).cuda()
    pos = torch.randint(0, 1 << 20, (n,), generator=gen).cuda()
    places = [slice(0, 1100), slice(n - 600, n)]
    outs = qk_norm_rotary_forward(q, k, w[0], w[1], pos)
    for at in places:
        few = qk_norm_rotary_forward(q[at], k[at], w[0], w[1], pos[at])
        assert all(torch.equal(a[at], b) for a, b in zip(outs, few))
    del outs
    # both gradients in the rows of one buffer, as those of a projection
    buf = torch.zeros((n, hq + hk + 1, d), dtype=BF16, device="cuda")
    qk_norm_rotary_backward(gq, gk, q, k, w[0], w[1], pos, into=(buf[:, :hq], buf[:, hq:hq + hk]))
    for at in places:
        few = qk_norm_rotary_backward(gq[at], gk[at], q[at], k[at], w[0], w[1], pos[at])
        assert torch.equal(buf[at, :hq], few[0]) and torch.equal(buf[at, hq:hq + hk], few[1])
    assert not buf[:, hq + hk:].any()
