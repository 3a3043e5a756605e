"""The table's gradient of very many tokens: up to the largest number of them, and long sums into one row."""
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
    # sums of 2,048 equal terms are exact; 2^20 of them are added up by fours and those in 64 bits: three roundings, and two of
    # the result
    assert abs(float(gw[0]) / (6.0 * (n - rare)) - 1) <= 5 * 2.0 ** -24


@pytest.mark.parametrize("v", [500, 2000])       # partial tables, sorted
@pytest.mark.parametrize("c", [4, 128, 1024, 1280])
def test_one_token_among_millions(v, c):
    # Equal rows, whose sums round to the same side at every addition.  float32: eight rows three additions deep, up to 192
    # such sums of a group of lanes (1,536 rows), the sums of up to 256 groups, and four roundings of what is added in 64 bits
    # (or six additions of 64 partial sums) and of the scale; more columns leave fewer groups: below 256 + 24 and 192 + 24
    from pymolecular_amd.embedding import embedding_backward
    n = 20_000_000 if c <= 128 else 2_000_000
    tokens = torch.full((n,), 7, device="cuda")
    tokens[::100_003] = v - 2
    few = (n + 100_002) // 100_003
    row = 1 + torch.rand((1, c), generator=torch.Generator().manual_seed(c)).cuda()
    gw = embedding_backward(row.expand(n, c), tokens, v, 0.3).double()
    want = torch.zeros((v, c), dtype=torch.float64, device="cuda")
    scale = float(torch.tensor(0.3))
    want[7], want[v - 2] = (n - few) * scale * row[0].double(), few * scale * row[0].double()
    err = ((gw - want).abs() / want.clamp(min=1e-30)).max()
    print(f"{float(err) * 2 ** 24:.1f} x 2^-24", flush=True)
    assert float(err) <= 290 * 2.0 ** -24
