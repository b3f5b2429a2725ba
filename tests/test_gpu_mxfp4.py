"""GPU tests of the microscaled 4-bit linear layers against their definition in 64 bits.

Tolerances.  Quantised operands are exact, and a product of two 4-bit values times powers of two is exact in fp32, so a sum of
K of them is off by at most K roundings of half a step, K 2^-24 times the sum of the terms' absolute values, whatever the
order; the bias and the residual add one rounding each.  A result rounded to bf16 adds 2^-8 of its value."""
import pytest
import torch

from laser_amd import _lib, grad_ops as G, ops, training
from mxfp4_ref import values

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
U32, UBF = 2.0 ** -24, 2.0 ** -8


def _x(rows, cols, dtype, scale=1.0):
    x = torch.randn(rows, cols, device="cuda") * scale
    return (x * (1 + 9 * (torch.rand(cols, device="cuda") < 0.05))).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 31), (2, 33), (64, 256), (65, 257), (130, 1000), (77, 512), (1, 4096)])
def test_quantize_is_the_definition(rows, cols, dtype):
    x = _x(rows, cols, dtype)
    q = ops.quantize_mxfp4(x)
    got = ops.dequantize_mxfp4(q)
    assert torch.equal(got.double(), values(x))
    t = ops.dequantize_mxfp4(q, transpose=True)
    assert t.shape == (cols, (rows + 63) // 64 * 64)
    assert torch.equal(t[:, :rows], got.t()) and not t[:, rows:].any()
    # a second quantisation changes nothing: every value of the format is its own nearest one unless the block's largest
    # element rounded down across a power of two, which the saturating end of the format excludes
    assert torch.equal(ops.dequantize_mxfp4(ops.quantize_mxfp4(got)), got)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quantize_strided_and_misaligned_rows(dtype):
    base = _x(40, 700, dtype)
    for view in (base[:, :512], base[:, 1:513], base[::2, 3:100], base[5:6, 7:8], base[:, :8].as_strided((40, 8), (700, 1), 4)):
        assert torch.equal(ops.dequantize_mxfp4(ops.quantize_mxfp4(view)).double(), values(view))


def test_quantize_every_bf16_value():
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF16).cuda()
    finite = every[torch.isfinite(every.float())]
    x = finite[torch.randperm(finite.numel(), device="cuda")][: finite.numel() // 32 * 32].view(-1, 32)
    assert torch.equal(ops.dequantize_mxfp4(ops.quantize_mxfp4(x)).double(), values(x))
    # sorted by magnitude: the blocks cover every exponent, the subnormal ones and zero among them
    x = finite[finite.float().abs().argsort()][: finite.numel() // 32 * 32].view(-1, 32)
    assert torch.equal(ops.dequantize_mxfp4(ops.quantize_mxfp4(x)).double(), values(x))


@pytest.mark.parametrize("top", [1.0, 1.9999999, 7.9e-38, 1.2e-38, 3e-39, 1e-40, 1.4e-45, 1.6e38])
def test_quantize_borders(top):
    """Every border between codes, its two neighbours and the block's maximum, at scales up to both ends of the range."""
    scale = 2.0 ** max(-127, torch.tensor(top, dtype=F64).log2().floor().item() - 2)
    marks = torch.tensor([0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7], dtype=F64) * scale
    near = marks.float()
    near = torch.cat([near, torch.nextafter(near, torch.tensor(0.0)), torch.nextafter(near, torch.tensor(1e38))])
    near = torch.cat([near[near <= top], torch.tensor([top])])
    x = torch.zeros(2 * near.numel(), 32)
    x[:, 0] = top
    x[: near.numel(), 5], x[near.numel():, 5] = near, -near
    x = x.cuda()
    assert torch.equal(ops.dequantize_mxfp4(ops.quantize_mxfp4(x)).double(), values(x).to(BF16).double())


def test_not_finite_blocks_read_back_as_nan():
    x = torch.zeros(4, 70, device="cuda")
    x[0, 3], x[1, 40], x[2, 69], x[3, 0] = float("nan"), float("inf"), float("-inf"), 3.0
    got = ops.dequantize_mxfp4(ops.quantize_mxfp4(x))
    want = torch.zeros(4, 70, dtype=torch.bool, device="cuda")
    want[0, :32], want[1, 32:64], want[2, 64:] = True, True, True
    assert torch.equal(torch.isnan(got), want) and got[3, 0] == 3.0


def _check(y, ref, size, K, terms, extra=0.0):
    """|y - ref| <= (K + terms) half steps of the absolute sum + extra."""
    bound = (K + terms) * U32 * size + extra + 1e-45
    worst = ((y.double() - ref).abs() - bound).max().item()
    assert worst <= 0, worst


SHAPES = [(1, 1, 1), (1, 64, 32), (3, 5, 33), (7, 1024, 4096), (16, 2048, 512), (17, 100, 300), (64, 64, 256), (65, 63, 255),
          (130, 257, 515), (300, 300, 1000), (1540, 768, 768), (2100, 2049, 640)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_against_64_bits(M, N, K, dtype):
    x, w = _x(M, K, dtype), 0.02 * torch.randn(N, K, device="cuda")
    b, r = torch.randn(N, device="cuda"), torch.randn(M, N, device="cuda")
    xv, wv = values(x), values(w)
    s, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    wq = ops.quantize_mxfp4(w)
    y = ops.linear_mxfp4(x, wq, b, residual=r)
    assert y.dtype == F32
    _check(y, r.double() + s + b.double(), size + b.double().abs() + r.double().abs(), K, 2)
    y = ops.linear_mxfp4(x, wq)
    assert y.dtype == BF16
    _check(y, s, size, K, 0, UBF * (s.abs() + K * U32 * size))
    # quick_gelu's slope is at most 1.1; its own few roundings are far below the bf16 one
    u = s + b.double()
    g = u * torch.sigmoid(1.702 * u)
    err = 1.1 * (K + 1) * U32 * (size + b.double().abs()) + 2.0 ** -20 * g.abs()
    _check(ops.linear_mxfp4(x, wq, b, gelu=True), g, 0 * size, 0, 0, err + UBF * (g.abs() + err))
    # operands quantised beforehand give the same sums
    _check(ops.linear_mxfp4(ops.quantize_mxfp4(x), wq, b, residual=r), r.double() + s + b.double(),
           size + b.double().abs() + r.double().abs(), K, 2)


@pytest.mark.parametrize("M,N,K", [(4200, 4100, 200), (4097, 4096, 512), (8192, 2560, 700), (16500, 1028, 1300), (33000, 512, 64)])
def test_linear_many_tiles(M, N, K):
    """More 256 x 256 tiles than compute units: several tiles per workgroup, ragged in both directions, one to six stages each."""
    x, w = _x(M, K, BF16), 0.02 * torch.randn(N, K, device="cuda")
    b, r = torch.randn(N, device="cuda"), torch.randn(M, N, device="cuda")
    xq, wq = ops.quantize_mxfp4(x), ops.quantize_mxfp4(w)
    xv, wv = values(x), values(w)
    s, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    y = ops.linear_mxfp4(xq, wq, b, residual=r)
    _check(y, r.double() + s + b.double(), size + b.double().abs() + r.double().abs(), K, 2)
    again = r.clone()
    assert torch.equal(ops.linear_mxfp4(x, wq, b, residual=again, out=again), y)
    _check(ops.linear_mxfp4(xq, wq), s, size, K, 0, UBF * (s.abs() + K * U32 * size))
    u = s + b.double()
    g = u * torch.sigmoid(1.702 * u)
    err = 1.1 * (K + 1) * U32 * (size + b.double().abs()) + 2.0 ** -20 * g.abs()
    y = ops.linear_mxfp4(xq, wq, b, gelu=True)
    _check(y, g, 0 * size, 0, 0, err + UBF * (g.abs() + err))
    for _ in range(3):
        assert torch.equal(ops.linear_mxfp4(xq, wq, b, gelu=True), y)


@pytest.mark.parametrize("M,N,K", [(2340, 4100, 200), (5000, 5004, 200), (4700, 4612, 512), (10300, 2564, 700), (20600, 1284, 1300),
                                   (66000, 516, 64), (4616, 1030, 768), (4600, 1028, 1100), (30000, 300, 40)])
def test_linear_every_kind_of_tile(M, N, K):
    """256 x 256 tiles in one round over the chip, in two and in four, ragged; 128 x 128 tiles with columns that allow wide accesses
    and with columns that do not."""
    test_linear_many_tiles(M, N, K)


@pytest.mark.parametrize("M,N,K", [(2340, 4099, 200), (5000, 5001, 200), (4700, 4614, 131), (20600, 1283, 1301), (66000, 517, 64), (4616, 1031, 767),
                                   (30000, 301, 40), (300, 131, 77), (90, 33, 1000), (20, 7, 31)])
def test_linear_of_any_alignment(M, N, K):
    """Odd row strides and column counts, operands that begin anywhere: every kernel, nothing written beside the result."""
    x = _x(M, K + 1, BF16)[:, 1:]
    w = 0.02 * torch.randn(N, K, device="cuda")
    b = torch.randn(N + 1, device="cuda")[1:]
    xv, wv = values(x), values(w)
    xq, wq = ops.quantize_mxfp4(x), ops.quantize_mxfp4(w)
    assert torch.equal(ops.dequantize_mxfp4(xq).double(), xv)
    s, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    store = torch.full((M + 2, N + 3), 7.0, device="cuda")
    out = store[1:-1, 1:1 + N]
    r = torch.randn(M, N, device="cuda")
    out.copy_(r)
    for q in (x, xq):
        out.copy_(r)
        ops.linear_mxfp4(q, wq, b, residual=out, out=out)
        _check(out, r.double() + s + b.double(), size + b.double().abs() + r.double().abs(), K, 2)
    u = s + b.double()
    g = u * torch.sigmoid(1.702 * u)
    err = 1.1 * (K + 1) * U32 * (size + b.double().abs()) + 2.0 ** -20 * g.abs()
    half = torch.full((M + 2, N + 3), 7.0, dtype=BF16, device="cuda")
    outh = half[1:-1, 1:1 + N]
    _check(ops.linear_mxfp4(xq, wq, b, gelu=True, out=outh), g, 0 * size, 0, 0, err + UBF * (g.abs() + err))
    _check(ops.linear_mxfp4(x, wq, out=outh), s, size, K, 0, UBF * (s.abs() + K * U32 * size))
    for t in (store, half):
        t[1:-1, 1:1 + N] = 7.0
        assert (t == 7.0).all()


def test_offsets_beyond_32_bits():
    """More than 2^32 elements: the last rows of each result are those of the last rows alone."""
    rows, cols, N = 1100000, 4000, 2048
    base = _x(997, cols, BF16)
    x = torch.empty((rows, cols), dtype=BF16, device="cuda")
    for at in range(0, rows, 997):
        x[at:at + 997] = base[: min(997, rows - at)]
    x[-64:] = _x(64, cols, BF16)
    tail = x[-64:].clone()
    q = ops.quantize_mxfp4(x)
    assert torch.equal(ops.dequantize_mxfp4(q)[-64:].double(), values(tail))
    sums, half = G.column_sums(x), x.new_zeros(cols, dtype=F64)
    for at in range(0, rows, 100000):
        half += x[at:at + 100000].sum(0, dtype=F64)
    assert (sums.double() - half).abs().max() <= 2.0 ** -16 * rows * base.abs().max().item()
    w = ops.quantize_mxfp4(0.02 * torch.randn(N, cols, device="cuda"))
    want = ops.linear_mxfp4(ops.quantize_mxfp4(tail), w, gelu=True)
    assert torch.equal(ops.linear_mxfp4(q, w, gelu=True)[-64:], want)
    assert torch.equal(ops.linear_mxfp4(x, w, gelu=True)[-64:], want)
    del q
    out = torch.empty((rows, N + 1), device="cuda")[:, 1:]          # rows that begin anywhere, in one kernel after another
    for n in (N, 1023):
        wn = w if n == N else ops.quantize_mxfp4(0.02 * torch.randn(n, cols, device="cuda"))
        o = out[:, :n]
        o.zero_()
        ops.linear_mxfp4(x, wn, residual=o, out=o)
        assert torch.equal(o[-64:], ops.linear_mxfp4(tail, wn, residual=torch.zeros(64, n, device="cuda")))


def test_linear_views_in_place_and_untouched_neighbours():
    M, N, K = 70, 96, 160
    x = _x(2 * M, K + 9, BF16)[::2, 5:5 + K]
    wq = ops.quantize_mxfp4(0.1 * torch.randn(N, K, device="cuda"))
    b = torch.randn(N, device="cuda")
    for rows in (M, 5):
        store = torch.full((rows + 2, N + 6), 7.0, device="cuda")
        r = store[1:1 + rows, 3:3 + N]
        r.copy_(torch.randn(rows, N, device="cuda"))
        want = ops.linear_mxfp4(x[:rows].contiguous(), wq, b, residual=r.clone())
        got = ops.linear_mxfp4(x[:rows], wq, b, residual=r, out=r)
        assert got.data_ptr() == r.data_ptr() and torch.equal(got, want)
        edge = store.clone()
        edge[1:1 + rows, 3:3 + N] = 7.0
        assert (edge == 7.0).all()


def test_not_finite_operands_reach_their_rows_and_columns_only():
    x, w = torch.randn(40, 96, device="cuda"), torch.randn(70, 96, device="cuda")
    x[3, 50], w[9, 1] = float("inf"), float("nan")
    want = torch.zeros(40, 70, dtype=torch.bool, device="cuda")
    want[3], want[:, 9] = True, True
    wq = ops.quantize_mxfp4(w)
    assert torch.equal(torch.isnan(ops.linear_mxfp4(x, wq)), want)
    assert torch.equal(torch.isnan(ops.linear_mxfp4(x[:10], wq)), want[:10])


def test_empty_and_zero():
    wq = ops.quantize_mxfp4(torch.randn(5, 64, device="cuda"))
    assert ops.linear_mxfp4(torch.empty(0, 64, device="cuda"), wq).shape == (0, 5)
    b = torch.randn(5, device="cuda")
    assert torch.equal(ops.linear_mxfp4(torch.zeros(40, 64, device="cuda"), wq, b), b.to(BF16).expand(40, 5))
    none = ops.quantize_mxfp4(torch.empty(0, 64, device="cuda"))
    assert ops.linear_mxfp4(torch.zeros(40, 64, device="cuda"), none).shape == (40, 0)


def test_refusals():
    x, w = torch.randn(4, 64, device="cuda"), ops.quantize_mxfp4(torch.randn(8, 64, device="cuda"))
    r, b = torch.randn(4, 8, device="cuda"), torch.randn(8, device="cuda")
    for bad in (lambda: ops.quantize_mxfp4(x.half()), lambda: ops.quantize_mxfp4(x[0]), lambda: ops.quantize_mxfp4(x.t()),
                lambda: ops.quantize_mxfp4(x.cpu()), lambda: ops.quantize_mxfp4(x[:, :0]), lambda: ops.quantize_mxfp4(x[:1].expand(4, 64)),
                lambda: ops.linear_mxfp4(x[:, :63], w), lambda: ops.linear_mxfp4(x, w, b[:7]), lambda: ops.linear_mxfp4(x, w, b.double()),
                lambda: ops.linear_mxfp4(x, w, gelu=True, residual=r), lambda: ops.linear_mxfp4(x, w, residual=r[:3]),
                lambda: ops.linear_mxfp4(x, w, residual=r.to(BF16)), lambda: ops.linear_mxfp4(x, w, out=r),
                lambda: ops.linear_mxfp4(x, w, residual=r, out=torch.empty(4, 9, device="cuda")),
                lambda: ops.linear_mxfp4(x, w, residual=r, out=x[:, :8]),
                lambda: ops.linear_mxfp4(x, w, residual=r[1:], out=r[:3]),
                lambda: ops.Mxfp4(w.data, 8, 300), lambda: ops.Mxfp4(w.data.float(), 8, 64), lambda: ops.Mxfp4(w.data[1:], 8, 64),
                lambda: training.linear_mxfp4(x, torch.randn(8, 63, device="cuda")),
                lambda: G.linear_mxfp4_bwd(r, ops.quantize_mxfp4(x), ops.quantize_mxfp4(x))):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    big = torch.randn(32, 64, device="cuda")
    y = torch.empty(32, 8, dtype=BF16, device="cuda")
    rc = lib.sgclip_mxfp4_linear(big.data_ptr(), 0, 64, w.codes.data_ptr(), w.scales.data_ptr(), 32, 8, 64, 0, None, None, 0, y.data_ptr(), 8,
                                 None, 0, st)
    assert rc == _lib.ENOSPC


def test_side_stream_and_replayed_graph():
    M, N, K = 200, 256, 320
    w, b = 0.1 * torch.randn(N, K, device="cuda"), torch.randn(N, device="cuda")
    x = torch.randn(M, K, device="cuda").to(BF16)
    want = ops.linear_mxfp4(x, ops.quantize_mxfp4(w), b, gelu=True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.linear_mxfp4(x, ops.quantize_mxfp4(w), b, gelu=True)
    side.synchronize()
    assert torch.equal(got, want)
    wq = ops.quantize_mxfp4(w)
    dy = torch.randn(M, N, device="cuda").to(BF16)

    def step():
        xq = ops.quantize_mxfp4(x)
        return ops.linear_mxfp4(x, wq, b, gelu=True), ops.linear_mxfp4(x[:3], wq, b), G.linear_mxfp4_bwd(dy, xq, wq)[0]
    for _ in range(2):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, c, dx = step()
    for k in range(4):
        x.copy_(torch.randn(M, K, device="cuda").to(BF16))
        graph.replay()
        torch.cuda.synchronize()
        ea, ec, edx = step()
        assert torch.equal(a, ea) and torch.equal(c, ec) and torch.equal(dx, edx), k


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,N", [(0, 5), (1, 1), (1, 512), (31, 513), (300, 77), (9000, 1032), (50, 8)])
def test_column_sums(M, N, dtype):
    x = _x(M, N + 3, dtype)[:, :N]
    for v in (x, x.contiguous()):
        got = G.column_sums(v)
        _check(got, v.double().sum(0), v.double().abs().sum(0), M, 0)
        assert torch.equal(G.column_sums(v), got)


def _grads_64(x, w, dy):
    xv, wv, d = values(x), values(w), dy.double()
    return d @ wv, d.t() @ xv, d.sum(0), (d.abs() @ wv.abs(), d.abs().t() @ xv.abs(), d.abs().sum(0))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,N,K", [(1, 64, 64), (5, 33, 77), (16, 8, 40), (385, 512, 512), (200, 100, 260), (64, 65, 257), (1200, 256, 768)])
def test_gradients_against_64_bits(M, N, K, dtype):
    x = _x(M, K, dtype).requires_grad_(True)
    w = (0.05 * torch.randn(N, K, device="cuda")).requires_grad_(True)
    b = torch.randn(N, device="cuda").requires_grad_(True)
    y = training.linear_mxfp4(x, w, b)
    assert torch.equal(y.detach(), ops.linear_mxfp4(ops.quantize_mxfp4(x.detach()), ops.quantize_mxfp4(w.detach()), b.detach()))
    dy = torch.randn(M, N, device="cuda").to(BF16)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    ex, ew, eb, (sx, sw, sb) = _grads_64(x.detach(), w.detach(), dy)
    assert dx.dtype == dtype and dw.dtype == F32 and db.dtype == F32
    # dy is bf16 already and the operands are exact: products of two bf16 values are exact in fp32
    _check(dx, ex, sx, N, 0, (UBF * (ex.abs() + N * U32 * sx)) if dtype == BF16 else 0.0)
    _check(dw, ew, sw, M, 0)
    _check(db, eb, sb, M, 0)


@pytest.mark.parametrize("M,N,K", [(513, 1032, 131), (1000, 517, 64), (9000, 96, 250)])
def test_gradients_of_f32_and_strided_dy(M, N, K):
    xq, wq = ops.quantize_mxfp4(_x(M, K, BF16)), ops.quantize_mxfp4(0.05 * torch.randn(N, K, device="cuda"))
    xv, wv = ops.dequantize_mxfp4(xq).double(), ops.dequantize_mxfp4(wq).double()
    for dy in (torch.randn(M, N, device="cuda"), torch.randn(M, N + 3, device="cuda")[:, 3:], torch.randn(M, N + 8, device="cuda").to(BF16)[:, 8:],
               torch.randn(M * N + 1, device="cuda").to(BF16)[1:].view(M, N)):
        d, r = dy.double(), dy.to(BF16).double()
        dx, dw, db = G.linear_mxfp4_bwd(dy, xq, wq, F32)
        _check(dx, r @ wv, r.abs() @ wv.abs(), N, 0)
        _check(dw, r.t() @ xv, r.abs().t() @ xv.abs(), M, 0)
        _check(db, d.sum(0), d.abs().sum(0), M, 0)
        for need in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
            got = G.linear_mxfp4_bwd(dy, xq, wq, F32, *need)
            assert [t is not None for t in got] == list(need)
            for t, whole in zip(got, (dx, dw, db)):
                assert t is None or torch.equal(t, whole) or (whole is dw and (t - dw).abs().max() <= 2 * M * U32 * (r.abs().t() @ xv.abs()).max())


def test_saved_operands_may_move():
    """Hooks that keep what forward saved elsewhere: backward finds it where they bring it back."""
    x, w = torch.randn(70, 96, device="cuda", requires_grad=True), torch.randn(40, 96, device="cuda", requires_grad=True)
    b = torch.randn(40, device="cuda", requires_grad=True)
    dy = torch.randn(70, 40, device="cuda").to(BF16)
    want = torch.autograd.grad(training.linear_mxfp4(x, w, b), (x, w, b), dy)
    with torch.autograd.graph.save_on_cpu():
        y = training.linear_mxfp4(x, w, b)
    for got, t in zip(torch.autograd.grad(y, (x, w, b), dy), want):
        assert torch.allclose(got, t, rtol=1e-5, atol=1e-5 * t.abs().max().item())


def test_gradients_against_differences():
    """y is linear in each quantised operand: a difference along any direction is the gradient's inner product exactly (64 bits)."""
    M, N, K = 40, 24, 96
    x, w = torch.randn(M, K, device="cuda"), 0.1 * torch.randn(N, K, device="cuda")
    dy = torch.randn(M, N, device="cuda").to(BF16)
    xq, wq = ops.quantize_mxfp4(x), ops.quantize_mxfp4(w)
    dx, dw, db = G.linear_mxfp4_bwd(dy, xq, wq, F32)
    loss = lambda a, c, e: ((a @ c.t() + e) * dy.double()).sum()  # noqa: E731
    xv, wv, bv = ops.dequantize_mxfp4(xq).double(), ops.dequantize_mxfp4(wq).double(), torch.zeros(N, dtype=F64, device="cuda")
    for grad, at in ((dx, 0), (dw, 1), (db, 2)):
        d = torch.randn(grad.shape, dtype=F64, device="cuda")
        args = [xv, wv, bv]
        up, down = list(args), list(args)
        up[at], down[at] = args[at] + d, args[at] - d
        slope = (loss(*up) - loss(*down)) / 2
        size = (grad.double().abs() * d.abs()).sum()
        assert (slope - (grad.double() * d).sum()).abs() <= max(M, N) * 2.0 ** -20 * size


def test_autograd_shapes_and_partial_gradients():
    x = torch.randn(2, 9, 64, device="cuda", requires_grad=True)
    w = torch.randn(32, 64, device="cuda")
    y = training.linear_mxfp4(x, w)
    assert y.shape == (2, 9, 32)
    y.sum().backward()          # an expanded gradient
    want = G.linear_mxfp4_bwd(torch.ones(18, 32, device="cuda", dtype=BF16), ops.quantize_mxfp4(x.detach().view(18, 64)), ops.quantize_mxfp4(w), F32)[0]
    assert torch.equal(x.grad.view(18, 64), want)
    wt = torch.randn(64, 32, device="cuda", requires_grad=True)
    training.linear_mxfp4(x.detach(), wt.t()).float().pow(2).sum().backward()
    assert wt.grad.shape == (64, 32) and torch.isfinite(wt.grad).all() and wt.grad.abs().sum() > 0
    with torch.no_grad():
        assert not training.linear_mxfp4(x, w).requires_grad


def test_autograd_of_empty_and_broadcast_operands():
    for M, N in ((0, 8), (5, 0), (0, 0)):
        x, w = torch.randn(M, 64, device="cuda", requires_grad=True), torch.randn(N, 64, device="cuda", requires_grad=True)
        b = torch.randn(N, device="cuda", requires_grad=True)
        training.linear_mxfp4(x, w, b).float().sum().backward()
        assert x.grad.shape == (M, 64) and w.grad.shape == (N, 64) and b.grad.shape == (N,)
        assert not x.grad.any() and not w.grad.any() and not b.grad.any()
    row, col = torch.randn(1, 64, device="cuda", requires_grad=True), torch.randn(1, 64, device="cuda", requires_grad=True)
    y = training.linear_mxfp4(row.expand(6, 64), col.expand(3, 64))
    dy = torch.randn(6, 3, device="cuda").to(BF16)
    y.backward(dy)
    dx, dw, _ = G.linear_mxfp4_bwd(dy, ops.quantize_mxfp4(row.detach().expand(6, 64).contiguous()), ops.quantize_mxfp4(col.detach().expand(3, 64).contiguous()), F32)
    assert torch.allclose(row.grad, dx.sum(0, keepdim=True), rtol=1e-5, atol=1e-5) and torch.allclose(col.grad, dw.sum(0, keepdim=True), rtol=1e-5, atol=1e-5)
    # strided x, and a transposed result's gradient
    wide = torch.randn(9, 2 * 64, device="cuda", requires_grad=True)
    w = torch.randn(16, 64, device="cuda")
    (training.linear_mxfp4(wide[:, ::2], w).t().float() * 2).sum().backward()
    assert not wide.grad[:, 1::2].any() and wide.grad[:, ::2].abs().sum() > 0


def test_autograd_is_refused_under_capture():
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    w = torch.randn(8, 64, device="cuda")
    training.linear_mxfp4(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="capture"):
            training.linear_mxfp4(x, w)
        y = training.linear_mxfp4(x.detach(), w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, training.linear_mxfp4(x.detach(), w))
