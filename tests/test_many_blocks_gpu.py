"""Layer norm and segment attention over more rows and segments than one launch has threads for: 2^32 threads, 2^20
workgroups at a time.

Every row of a norm, and every segment, is by itself, so the result at the places where launches meet and end is that of
a call on a few of them, bit for bit.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


def _places(n, part):
    """Ranges of rows at the start, at the end and around every boundary between parts."""
    for at in range(0, n, part):
        yield slice(max(0, at - 40), min(n, at + 40))
    yield slice(n - 50, n)


def _fill(*shape, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)


# two columns: four lanes a row, 2^32 threads at 2^30 rows; rows past a wave's registers: a workgroup each
@pytest.mark.parametrize("n,c,dtype,part", [((1 << 30) + 77, 2, BF16, 1 << 26), ((1 << 26) + 5, 3, F32, 1 << 26),
                                            ((1 << 20) + 3, 1541, F32, 1 << 20)])
def test_norm_forward(n, c, dtype, part):
    from pymolecular_amd.layer_norm import layer_norm, layer_norm_forward
    x = _fill(n, c, dtype=dtype, seed=c)
    w, b = _fill(c, dtype=dtype, seed=1), _fill(c, dtype=dtype, seed=2)
    y = layer_norm(x, w, b)
    for i in _places(n, part):
        assert torch.equal(y[i], layer_norm(x[i].contiguous(), w, b)), i
    del y
    if c != 2:
        r = _fill(n, c, dtype=dtype, seed=3)
        out = layer_norm_forward(x, w, b, residual=r)
        for i in _places(n, part):
            for p, q in zip(out, layer_norm_forward(x[i].contiguous(), w, b, residual=r[i].contiguous())):
                assert torch.equal(p[i], q), i


def test_norm_backward_of_wide_rows():
    from pymolecular_amd.layer_norm import layer_norm_backward, layer_norm_forward
    n, c = (1 << 20) + 3, 1541
    x, gy = _fill(n, c, dtype=F32, seed=4), _fill(n, c, dtype=F32, seed=5)
    w = _fill(c, dtype=F32, seed=1)
    y, s, mean, rstd = layer_norm_forward(x, w)
    del y
    gx, gw, gb = layer_norm_backward(gy, s, w, mean, rstd, gsum=x)
    for i in _places(n, 1 << 20):
        small = layer_norm_backward(gy[i].contiguous(), s[i].contiguous(), w, mean[i].contiguous(), rstd[i].contiguous(),
                                    gsum=x[i].contiguous())
        assert torch.equal(gx[i], small[0]), i
    # gb: 128 fp32 sums of 2^13 values of about 1, each addition rounding a sum of about 2^6.5: 2^-24 2^6.5 2^6.5 a sum and
    # 2^3.5 times that for all of them; four deviations, for 1,541 columns, and a half for the addition of the 128
    want = sum(g.double().sum(dim=0) for g in gy.split(1 << 17))
    assert (gb.double() - want).abs().max() <= 2.0 ** -24 * 2.0 ** 16.5 * 4.5


# segments of `rows` rows.  A wave a segment and four a workgroup, 2^32 threads at 2^26 of them; two waves a segment; waves
# with tiles of heads wider than 64; workgroups with tiles of 64 rows
@pytest.mark.parametrize("n,rows,d,dtype,part", [((1 << 26) + 9, 2, 8, BF16, 1 << 22), ((1 << 20) + 5, 2, 8, F32, 1 << 20),
                                                 ((1 << 21) + 7, 2, 72, BF16, 1 << 21), ((1 << 20) + 5, 2, 72, F32, 1 << 20),
                                                 ((1 << 20) + 5, 30, 16, BF16, 1 << 20)])
def test_attention(n, rows, d, dtype, part):
    from pymolecular_amd.segment_attention import segment_attention_backward, segment_attention_forward
    x = [_fill(n * rows, 1, d, dtype=dtype, seed=i) for i in range(4)]
    ptr = torch.arange(0, n * rows + 1, rows, dtype=torch.int32, device="cuda")
    out, lse = segment_attention_forward(*x[:3], ptr)
    grads = segment_attention_backward(x[3], *x[:3], out, lse, ptr)
    for i in _places(n, part):
        j = slice(i.start * rows, i.stop * rows)
        few = [t[j].contiguous() for t in x]
        p = ptr[:i.stop - i.start + 1].contiguous()
        o, l = segment_attention_forward(*few[:3], p)
        for a, b in zip((out[j], lse[:, j], *(g[j] for g in grads)), (o, l, *segment_attention_backward(few[3], *few[:3], o, l, p))):
            assert torch.equal(a, b), i


def test_counts_past_32_bits_are_refused():
    # 2^32 + 5 columns are not 5 columns, 2^32 + 1 segments not one
    from pymolecular_amd.layer_norm import layer_norm
    from pymolecular_amd.segment_attention import segment_attention
    wide = torch.zeros((1, (1 << 32) + 5), dtype=BF16, device="cuda")
    with pytest.raises(ValueError):
        layer_norm(wide)
    del wide
    ptr = torch.zeros((1 << 32) + 2, dtype=torch.int32, device="cuda")
    ptr[-1] = 20
    x = _fill(20, 2, 16, dtype=BF16, seed=0)
    with pytest.raises(ValueError):
        segment_attention(x, x, x, ptr)
    del ptr
    many = torch.zeros((0, (1 << 32) + 2, 16), dtype=BF16, device="cuda")
    with pytest.raises(ValueError):
        segment_attention(many, x[:0], x[:0], torch.zeros(2, dtype=torch.int32, device="cuda"))
