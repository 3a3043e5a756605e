"""The table's gradient at the largest number of tokens, 2^31 - 1."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rare", [200, 700])
def test_most_tokens(rare):
    # sorted, with the last table row's few tokens at the very end of the order
    from pymolecular_amd.embedding import embedding_backward
    n, v = (1 << 31) - 1, 20000
    tokens = torch.zeros(n, dtype=torch.int32, device="cuda")
    tokens[5:5 + rare] = v - 1
    gw = embedding_backward(torch.full((1, 1), 3.0, device="cuda").expand(n, 1), tokens, v, 2.0)
    assert float(gw[v - 1]) == 6.0 * rare and not gw[1:v - 1].any()
    # sums of 2,048 equal terms are exact; 2^20 of them are added in turn by 256 groups, and those then: a rounding each
    assert abs(float(gw[0]) / (6.0 * (n - rare)) - 1) <= (4096 + 256) * 2.0 ** -24
