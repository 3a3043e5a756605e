"""Forms of segment attention, layer norm and the network of both that the other tests do not reach: small segments of
heads wider than 64, statistics of the stored sum in rows of every kernel, other widths and batches of the network.

Bounds are those of the modules whose comparisons are used here.  The norm's gradients are compared with the formulas at the
sum as it is stored, from which they are made: one rounding of the result, 2 x 2^-9 as in test_layer_norm_gpu.py.
"""
import numpy as np
import pytest
import torch

import test_global_attention_gpu as net
from oracle import attention_ref as ref
from test_segment_attention_gpu import _case, _compare

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16

# waves with tiles of 16 rows (up to 28 rows a segment), heads of 65 to 128 values
SHORT_WIDE = [([20, 3, 32, 33, 1, 0, 7] + [11] * 40, None, 4, 2, 96), ([9, 29, 17, 1, 2, 16], None, 4, 4, 128),
              ([8] * 30 + [40], [20] * 30 + [90], 4, 1, 72), ([1] * 70, [19] * 35 + [23] * 35, 8, 2, 128),
              ([12, 0, 9, 16, 17, 31], [9, 20, 0, 16, 90, 2], 6, 2, 104)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("lq,lk,hq,hk,d", SHORT_WIDE)
def test_short_segments_of_wide_heads(dtype, masked, lq, lk, hq, hk, d):
    q, k, v, go, a, b = _case(lq, lk, hq, hk, d, dtype, seed=d + hq, lead=4, tail=50, packed=lk is None)
    mask = torch.rand(k.shape[0], generator=torch.Generator().manual_seed(3)).cuda() < 0.6 if masked else None
    _compare(q, k, v, go, a, b, mask)


def _rel(a, b):
    a = a.detach().double().cpu().numpy()
    return np.linalg.norm(a - b) / np.linalg.norm(b)


@pytest.mark.parametrize("offset", [4.0, 300.0])
@pytest.mark.parametrize("n,c", [(40, 128), (40, 99), (30, 2500), (20, 12289), (70000, 42)])
def test_statistics_of_the_stored_sum(n, c, offset):
    # rows whose mean exceeds their deviation, in bf16: at 300 the sum is stored in steps of 2 deviations
    from pymolecular_amd.layer_norm import layer_norm_backward, layer_norm_forward
    gen = torch.Generator().manual_seed(c)
    rand = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    x, r = rand(n, c).to(BF16).cuda(), (offset * (1 + 0.1 * rand(n, 1)) + 0 * rand(1, c)).expand(n, c).to(BF16).cuda()
    w, gy, gs = (1 + 0.2 * rand(c)).to(BF16).cuda(), rand(n, c).to(BF16).cuda(), rand(n, c).to(BF16).cuda()
    y, s, mean, rstd = layer_norm_forward(x, w, residual=r)
    assert torch.equal(s, x + r)
    np64 = lambda t: t.double().cpu().numpy()  # noqa: E731
    got = layer_norm_backward(gy, s, w, mean, rstd, gs)
    want = ref.layer_norm_grads_ref(np64(gy), np64(s), np64(w), 1e-5, np64(gs))
    errs = [_rel(y, ref.layer_norm_ref(np64(x), np64(w), None, 1e-5, np64(r))[0])] + [_rel(a, b) for a, b in zip(got, want)]
    print([f"{e:.1e}" for e in errs], flush=True)
    # where |mean| is near the deviation the kept statistics may be those of the unrounded sum: 2^-9 |mean| / std of it in xh
    assert max(errs) <= 2 * 2.0 ** -9


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype,tol", [(F32, 5e-5), (BF16, 6e-2)])
@pytest.mark.parametrize("width,heads,kv_heads,graphs", [(256, 2, 1, 5), (128, 8, 1, 3), (128, 4, 4, 40)])
def test_network_of_other_widths(monkeypatch, width, heads, kv_heads, graphs, dtype, tol, masked):
    batch = net.graphs.molecule_batch
    for name, value in (("H", width), ("HEADS", heads), ("KV", kv_heads)):
        monkeypatch.setattr(net, name, value)
    monkeypatch.setattr(net.graphs, "molecule_batch", lambda n, **kw: batch(graphs, **kw))
    net.test_network_matches_float64(dtype, tol, masked)


def test_a_width_without_message_kernels_is_refused(monkeypatch):
    # layers of 64 features and 64 messages have no kernels: an error, whatever follows them
    monkeypatch.setattr(net, "H", 64)
    with pytest.raises(ValueError, match="unsupported dimensions"):
        net.test_network_matches_float64(F32, 5e-5, False)
