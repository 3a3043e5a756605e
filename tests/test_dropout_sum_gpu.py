"""What layer norm behind a dropout keeps beside a bfloat16 sum, against the sum itself.

The sum is made in float32 from x up and the residual, two roundings (2^-23 of it and of x up at most).  What the bfloat16
rounding takes from it or adds is up to 32,768 units in the last place of float32 (2^-23 of the value's power of two).  The int16
gives all of them back, but for one where 32,768 were taken.  The int8 gives back steps of 256, to half a step, and 127 of them
where more were taken: 256 units are left of 32,768.
"""
import numpy as np
import pytest
import torch

from oracle.dropout_ref import dropout_ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _sums(c):
    """x and the residual (n, c) in bfloat16: all pairs of a value of [1, 2) and a multiple of 2^-15 below 2^-7, half-way sums
    of both parities among them, of either sign."""
    x, r = (1 + torch.arange(128) * 2.0 ** -7).repeat_interleave(256), (torch.arange(256) * 2.0 ** -15).repeat(128)
    return (torch.cat([t, -t]).to(BF16).view(-1, c).cuda() for t in (x, r))


@pytest.mark.parametrize("params", [F32, BF16])
@pytest.mark.parametrize("c", [64, 4096])       # rows in a wave's registers, and past them
def test_what_the_rounding_lost(c, params):
    from pymolecular_amd.dropout import Dropout
    from pymolecular_amd.layer_norm import layer_norm_dropout_forward
    rng = torch.tensor([3, 4], device="cuda")
    x, r = _sums(c)
    lows = set()
    for p, small in ((0.0, r), (0.3, r), (0.3, x * 0.37)):
        w = torch.ones(c, dtype=params, device="cuda")
        y, s, mean, (rstd, low) = layer_norm_dropout_forward(x, small, Dropout(p, rng), w)
        assert low.dtype == (torch.int16 if params == F32 else torch.int8)
        scaled = dropout_ref(x.double().cpu().numpy(), p, 3, 4)
        want = scaled + small.double().cpu().numpy()
        step = 1 if params == F32 else 256
        got = (s.float().view(torch.int32) + step * low.to(torch.int32)).view(F32).double().cpu().numpy()
        unit = 2.0 ** (np.floor(np.log2(np.abs(want) + 1e-300)) - 23)
        err = np.abs(got - want) - 2.0 ** -23 * (np.abs(want) + np.abs(scaled))
        most = 1 if params == F32 else np.where(low.cpu().numpy() == 127, 256, 128)
        assert (err <= most * unit).all(), (err / unit).max()
        lows |= set(low.unique().tolist())
    assert (min(lows), max(lows)) == ((-32768, 32767) if params == F32 else (-128, 127))
