"""CPU tests of the 4-bit linear layers' host side: storage sizes, and arguments that are refused before any launch."""
import pytest
import torch

from laser_amd import _lib, ops, training
from mxfp4_ref import values


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__ as g
        g.build()
    return _lib.load()


def test_storage_sizes(lib):
    assert lib.sgclip_mxfp4_codes_bytes(3, 257) == 3 * 256 and lib.sgclip_mxfp4_scales_bytes(3, 257) == 64 * 16
    assert lib.sgclip_mxfp4_codes_bytes(65, 256) == 65 * 128 and lib.sgclip_mxfp4_scales_bytes(65, 256) == 128 * 8
    assert lib.sgclip_mxfp4_codes_bytes(0, 256) == 0 and lib.sgclip_mxfp4_scales_bytes(-1, 5) == 0
    assert lib.sgclip_mxfp4_codes_bytes(1 << 22, 4096) == (1 << 22) * 2048          # beyond 32 bits
    assert lib.sgclip_mxfp4_linear_workspace_bytes(16, 4096) == 0
    assert lib.sgclip_mxfp4_linear_workspace_bytes(17, 256) == 17 * 128 + 128 + 64 * 8   # codes rounded up to a multiple of 256, scales


def test_python_storage_sizes_agree(lib):
    for rows in (0, 1, 63, 64, 65, 1000, 1 << 20):
        for cols in (1, 32, 255, 256, 257, 4096):
            assert ops.Mxfp4.sizes(rows, cols) == (lib.sgclip_mxfp4_codes_bytes(rows, cols), lib.sgclip_mxfp4_scales_bytes(rows, cols))


def test_entry_points_refuse_bad_arguments(lib):
    p = 4096  # an aligned address that no refused call touches
    E = _lib.EINVAL
    assert lib.sgclip_mxfp4_quantize(p, 0, 8, 0, 8, p, p, None) == _lib.OK          # no rows: nothing to do
    for rows, cols, ldx, dtype, c in ((-1, 8, 8, 0, p), (4, 0, 8, 0, p), (4, 8, 7, 0, p), (4, 8, 8, 2, p), (4, 8, 8, 0, p + 8), (4, 8, 8, 0, None),
                                      ((1 << 30) + 1, 8, 8, 0, p), (4, (1 << 24) + 1, 1 << 25, 0, p), (1 << 30, 1 << 16, 1 << 16, 0, p)):
        assert lib.sgclip_mxfp4_quantize(p, dtype, ldx, rows, cols, c, p, None) == E
        assert lib.sgclip_last_error()
    assert lib.sgclip_mxfp4_quantize(None, 0, 8, 4, 8, p, p, None) == E
    for tr, ldo in ((0, 7), (1, 3), (1, 65)):
        assert lib.sgclip_mxfp4_dequantize(p, p, 4, 8, tr, p, ldo, None) == E
    assert lib.sgclip_mxfp4_dequantize(p, p, 1 << 30, 1 << 16, 0, p, 1 << 16, None) == E
    ok = dict(xc=p, xs=p, wc=p, ws=p, M=4, N=8, K=32, epi=0, bias=None, aux=None, lda=0, out=p, ldo=8)

    def gemm(**kw):
        a = dict(ok, **kw)
        return lib.sgclip_mxfp4_gemm(*(a[k] for k in ("xc", "xs", "wc", "ws", "M", "N", "K", "epi", "bias", "aux", "lda", "out", "ldo")), None)
    for bad in (dict(xc=None), dict(ws=p + 4), dict(K=0), dict(M=-1), dict(epi=_lib.EPI_F32), dict(out=None), dict(ldo=7),
                dict(epi=_lib.EPI_BIAS_RESID_F32), dict(epi=_lib.EPI_BIAS_RESID_F32, aux=p, lda=7), dict(M=1 << 30, N=1 << 20, ldo=1 << 20)):
        assert gemm(**bad) == E, bad
    assert gemm(M=0) == _lib.OK and gemm(N=0) == _lib.OK
    assert lib.sgclip_mxfp4_linear(p, 0, 32, p, p, 17, 8, 32, 0, None, None, 0, p, 8, p, 16, None) == _lib.ENOSPC
    assert lib.sgclip_mxfp4_linear(p, 0, 31, p, p, 4, 8, 32, 0, None, None, 0, p, 8, None, 0, None) == E
    assert lib.sgclip_mxfp4_linear(p, 5, 32, p, p, 4, 8, 32, 0, None, None, 0, p, 8, None, 0, None) == E


def test_host_tensors_are_refused(lib):
    with pytest.raises(ValueError, match="GPU"):
        ops.quantize_mxfp4(torch.zeros(4, 32))
    with pytest.raises(ValueError):
        ops.Mxfp4(torch.zeros(4 * 128 + 64 * 8, dtype=torch.uint8), 4, 32)
    with pytest.raises(ValueError, match="fit"):
        training.linear_mxfp4(torch.zeros(4, 32), torch.zeros(8, 31))


def test_reference_values():
    """The definition the GPU tests compare with, on values worked out by hand: block maximum 4 has scale 1."""
    x = torch.zeros(1, 40)
    x[0, :16] = torch.tensor([4.0, 0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, -0.75, 3.49, 2.51, 0.24, -3.5, 1.0, 3.0, 0.5])
    x[0, 32:34] = torch.tensor([7.0, 5.0])
    want = [4, 0, 0.5, 1, 1, 2, 2, 4, -1, 3, 3, 0, -4, 1, 3, 0.5]
    got = values(x)
    assert got[0, :16].tolist() == want and got[0, 32:34].tolist() == [6, 4]


def test_gradient_entry_point(lib):
    p, E = 4096, _lib.EINVAL
    need = lib.sgclip_mxfp4_linear_bwd_workspace_bytes
    # zeros [K], w^T [K][64], x [M][K]; what has to be laid out or cropped comes on top
    plain = 256 + 64 * 64 * 2 + 40 * 64 * 2
    assert need(p, _lib.DTYPE_BF16, 64, 40, 64, 64) == plain
    for dy, dtype, ld in ((p, _lib.DTYPE_F32, 64), (p + 8, _lib.DTYPE_BF16, 64), (p, _lib.DTYPE_BF16, 68)):
        assert need(dy, dtype, ld, 40, 64, 64) == plain + 40 * 64 * 2
    assert need(p, _lib.DTYPE_BF16, 61, 40, 61, 64) == plain + 40 * 64 * 2 + 64 * 64 * 4
    assert need(p, _lib.DTYPE_BF16, 64, 1000, 64, 64) == 256 + 64 * 64 * 2 + 1000 * 64 * 2 + 32 * 64 * 4     # strips of column sums
    assert need(p, _lib.DTYPE_BF16, 64, 0, 64, 64) == need(p, _lib.DTYPE_BF16, 0, 5, 0, 64) == 0

    def bwd(dy=p, dtype=_lib.DTYPE_BF16, ld=64, xc=p, ws=p, M=40, N=64, K=64, dx=p, dxt=_lib.DTYPE_BF16, dw=p, work=p, size=1 << 20):
        return lib.sgclip_mxfp4_linear_bwd(dy, dtype, ld, xc, p, p, ws, M, N, K, dx, dxt, dw, p, work, size, None)
    for bad in (dict(dy=None), dict(dtype=7), dict(ld=63), dict(xc=None), dict(ws=p + 4), dict(M=-1), dict(K=0), dict(dxt=7)):
        assert bwd(**bad) == E and lib.sgclip_last_error(), bad
    for bad in (dict(work=None), dict(work=p + 8), dict(size=100)):
        assert bwd(**bad) == _lib.ENOSPC
