"""What GlobalAttention and EGNNGlobal refuse when they are built, without a GPU."""
import pytest

from pymolecular_amd.models.EGNN import EGNNGlobal, GlobalAttention


@pytest.mark.parametrize("hidden,heads", [(60, 4), (6, 2), (5, 5), (260, 2), (512, 2)])
def test_head_widths_that_cannot_be_normed(hidden, heads):
    # odd, or wider than 128: every forward would raise
    for build in (lambda: GlobalAttention(hidden, heads, qk_norm=True), lambda: EGNNGlobal(4, hidden, 1, heads=heads, qk_norm=True)):
        with pytest.raises(ValueError, match="qk_norm.*%d.*%d" % (hidden, heads)):
            build()
    GlobalAttention(hidden, heads)            # (the attention alone takes odd widths)


@pytest.mark.parametrize("hidden,heads", [(60, 5), (256, 2), (2, 1), (128, 4)])
def test_head_widths_that_can(hidden, heads):
    assert GlobalAttention(hidden, heads, qk_norm=True).q_weight.shape == (hidden // heads,)
