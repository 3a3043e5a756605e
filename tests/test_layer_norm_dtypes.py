"""Parameter dtype of the layer norm's C entries, without a GPU."""
from pymolecular_amd import _capi

BUF = 1 << 12   # a non-NULL aligned stand-in address, never dereferenced by the calls below


def test_float32_parameters_are_checked():
    L = _capi.lib()
    dims = lambda f: _capi.EgnnNormDims(10, 64, 1, 1e-5, f)  # noqa: E731
    fwd = lambda f, w=BUF, b=BUF, eps=1e-5: L.egnn_norm_fwd(dims(f), BUF, 64, None, 0, w, b, BUF, None, BUF, BUF, None)  # noqa: E731
    assert fwd(2) == fwd(-1) == _capi.EGNN_ERR_DIMS and L.egnn_norm_bwd_workspace_bytes(dims(2)) == 0
    assert fwd(1, w=BUF + 2) == fwd(1, b=BUF + 2) == 4 == fwd(0, w=BUF + 1)     # aligned to their own dtype
    bwd = lambda f, w=BUF, gw=BUF, gb=BUF: L.egnn_norm_bwd(dims(f), BUF, 64, BUF, 64, w, BUF, BUF, None, 0, BUF, gw, gb, None, 0, None)  # noqa: E731
    assert bwd(1, w=BUF + 2) == bwd(1, gw=BUF + 2) == bwd(1, gb=BUF + 2) == 4
    assert bwd(0, w=BUF + 2, gw=BUF + 2, gb=BUF + 2) == bwd(1) == 5              # asks for the workspace next
