"""CPU tests of the 4-bit layer's gradients' limits: what is laid out anew, and what is refused before anything is written."""
import os

import pytest

from laser_amd import _lib


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__ as g
        g.build()
    return _lib.load()


def test_row_strides_that_the_products_cannot_take_are_laid_out(lib):
    need = lib.sgclip_mxfp4_linear_bwd_workspace_bytes
    p, M, N, K = 4096, 40, 64, 64
    plain = need(p, _lib.DTYPE_BF16, N, M, N, K)
    assert need(p, _lib.DTYPE_BF16, 1 << 22, M, N, K) == plain
    for ld in ((1 << 22) + 8, 1 << 25, 1 << 40):         # 256 rows of them pass what the products' 32-bit offsets hold
        assert need(p, _lib.DTYPE_BF16, ld, M, N, K) == plain + M * 64 * 2


def test_more_columns_than_the_products_take(lib):
    p = 4096
    for n, rc in (((1 << 22) + 1, _lib.EINVAL), (1 << 24, _lib.EINVAL), (1 << 22, _lib.ENOSPC)):
        assert lib.sgclip_mxfp4_linear_bwd(p, _lib.DTYPE_BF16, n, p, p, p, p, 4, n, 64, p, _lib.DTYPE_BF16, p, p, p, 100, None) == rc
        assert lib.sgclip_last_error()
