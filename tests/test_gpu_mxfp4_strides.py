"""GPU tests of the 4-bit layer's gradients for a dy whose rows lie apart: read where they are, with the bits of a dy in one piece."""
import pytest
import torch

from laser_amd import grad_ops as G, ops

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def views(M, N):
    """Row strides that the products take as they are, and ones that are laid out for them; a stride that no copy keeps."""
    wide = torch.randn(M, 2 * N + 24, device="cuda")
    yield "aligned", wide.to(BF16)[:, 8:8 + N]
    yield "odd start", wide.to(BF16)[:, 3:3 + N]
    yield "f32", wide[:, 1:1 + N]
    yield "every other row", torch.randn(2 * M, N, device="cuda").to(BF16)[::2]
    yield "odd stride", torch.randn(M, N + 1, device="cuda").to(BF16)[:, :N]
    yield "one row", torch.randn(1, N, device="cuda").to(BF16).expand(M, N)
    yield "transposed", torch.randn(N, M, device="cuda").to(BF16).t()


@pytest.mark.parametrize("M,N,K", [(700, 256, 192), (300, 100, 72), (1, 64, 64), (130, 1, 40), (1, 1, 33), (5000, 512, 256)])
def test_strided_rows(M, N, K):
    xq, wq = ops.quantize_mxfp4(torch.randn(M, K, device="cuda")), ops.quantize_mxfp4(0.05 * torch.randn(N, K, device="cuda"))
    xv = ops.dequantize_mxfp4(xq).double()
    for name, dy in views(M, N):
        dx, dw, db = G.linear_mxfp4_bwd(dy, xq, wq, F32)
        ex, ew, eb = G.linear_mxfp4_bwd(dy.contiguous().clone(), xq, wq, F32)
        assert torch.equal(dx, ex) and torch.equal(db, eb), name
        # fp32 atomics in another order: M roundings of half a step, on either side
        assert ((dw - ew).abs().double() <= 2 * M * 2.0 ** -24 * (dy.double().abs().t() @ xv.abs())).all(), name


def test_strided_rows_are_not_copied():
    M, N, K = 20000, 1024, 64
    xq, wq = ops.quantize_mxfp4(torch.randn(M, K, device="cuda")), ops.quantize_mxfp4(0.05 * torch.randn(N, K, device="cuda"))
    peaks = []
    for dy in (torch.randn(M, N, device="cuda").to(BF16), torch.randn(M, 2 * N, device="cuda").to(BF16)[:, N:]):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        G.linear_mxfp4_bwd(dy, xq, wq)
        torch.cuda.synchronize()
        peaks.append(torch.cuda.max_memory_allocated() - before)
    assert peaks[1] <= peaks[0] + M * N      # half of a copy


def test_a_row_stride_beyond_the_products_offsets():
    M, N, K = 300, 64, 64
    ld = (1 << 23) + 8                       # 16 MB from row to row: 256 of them pass 32 bits
    store = torch.empty(M * ld, dtype=BF16, device="cuda")
    dy = store.as_strided((M, N), (ld, 1))
    dy.copy_(torch.randn(M, N, device="cuda"))
    xq, wq = ops.quantize_mxfp4(torch.randn(M, K, device="cuda")), ops.quantize_mxfp4(0.05 * torch.randn(N, K, device="cuda"))
    dx, dw, db = G.linear_mxfp4_bwd(dy, xq, wq, F32)
    ex, ew, eb = G.linear_mxfp4_bwd(dy.contiguous(), xq, wq, F32)
    assert torch.equal(dx, ex) and torch.equal(db, eb) and torch.allclose(dw, ew, rtol=1e-4, atol=1e-3)
    del store, dy
    torch.cuda.empty_cache()
