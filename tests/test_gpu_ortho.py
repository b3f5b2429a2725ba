"""GPU tests of the orthogonalised updates against the iteration in 64 bits.

Tolerances, relative in the Frobenius norm.  An operand is held in 22 bits (two fp16 halves: off by 2^-23 of its value at most), sums
in fp32.  With p(t) = a + b t + c t^2 and |X| = 1 at the start:
  step by step, a rounding of X (and of p(A) X, which is one) grows by at most a per remaining step: about four roundings in each
  of five steps, each at most 2^-23 a^5 in the result whose norm is |O|;
  as one block, a rounding of A (at most 2^-23 of its norm, at most 1) shifts small eigenvalues, and with them the product P of the five
  polynomials by P'(0) / P(0) = (b / a) (1 + a^2 + a^4 + a^6 + a^8) = 3e4 of itself: 3.6e-3.
A bf16 result is off by another 2^-8 of each element."""
import math

import pytest
import torch
from torch import nn

from laser_amd import grad_ops as G, ops, training

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
A, B, C2 = G.NEWTON_SCHULZ
UBF, U32 = 2.0 ** -8, 2.0 ** -24
BLOCK = abs(B) / A * sum(A ** (2 * k) for k in range(5)) * 2.0 ** -23
SINGLE = 20 * A ** 5 * 2.0 ** -23


def iterate(g, steps=5, coefficients=G.NEWTON_SCHULZ, eps=1e-7):
    x = g.double()
    flip = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2).contiguous() if flip else x
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + eps)
    table = coefficients if isinstance(coefficients[0], (tuple, list)) else [coefficients] * steps
    for a, b, c in table:
        gram = x @ x.transpose(-1, -2).contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-1, -2).contiguous() if flip else x


def rel(x, y):
    return ((x.double() - y).norm() / y.norm()).item()


def tolerance(rows, cols, o):
    m, n = min(rows, cols), max(rows, cols)
    single = n * 4 < m * 5 or m < 256
    return SINGLE / o.norm().item() + 2.0 ** -20 if single else BLOCK


def spectrum(kind, rows, cols, batch=1):
    m = min(rows, cols)
    if kind == "gaussian":
        return torch.randn(batch, rows, cols, device="cuda")
    if kind == "low rank":        # exactly: most singular values are zero
        k = max(1, m // 8)
        return torch.randn(batch, rows, k, device="cuda") @ torch.randn(batch, k, cols, device="cuda")
    if kind == "strong directions":
        k = min(8, m)
        return torch.randn(batch, rows, k, device="cuda") @ torch.randn(batch, k, cols, device="cuda") + 0.02 * torch.randn(batch, rows, cols, device="cuda")
    u = torch.linalg.qr(torch.randn(batch, rows, m, dtype=F64))[0]
    v = torch.linalg.qr(torch.randn(batch, cols, m, dtype=F64))[0]
    s = torch.exp(-8 * torch.arange(m, dtype=F64) / m)
    return ((u * s) @ v.transpose(1, 2)).float().cuda()


def raw(g, **kw):
    """The result before its rounding to bf16: a step from zero parameters with rate -1, without momentum."""
    g3 = g if g.dim() == 3 else g[None]
    p, buf = torch.zeros(g3.shape, device="cuda"), torch.zeros(g3.shape, device="cuda")
    G.muon_step(list(p), list(g3.float().contiguous()), buf, lr=-1.0, momentum=0.0, nesterov=False, **kw)
    return p if g.dim() == 3 else p[0]


SHAPES = [(1, 1, 1), (2, 1, 40), (3, 40, 1), (2, 33, 20), (2, 127, 255), (1, 64, 64), (3, 130, 129), (2, 65, 31), (1, 300, 700), (2, 700, 300),
          (1, 257, 256), (1, 768, 768), (1, 512, 2048), (30, 200, 300), (70, 48, 32), (16, 256, 1000)]


@pytest.mark.parametrize("kind", ["gaussian", "strong directions"])
@pytest.mark.parametrize("batch,rows,cols", SHAPES)
def test_against_64_bits(batch, rows, cols, kind):
    g = 1e-3 * spectrum(kind, rows, cols, batch)
    want = iterate(g)
    got, tol = raw(g), tolerance(rows, cols, want / math.sqrt(batch))
    assert rel(got, want) <= tol
    for dtype in (F32, BF16):
        x = g.to(dtype)
        want = iterate(x)
        y = G.orthogonalize(x)
        assert y.dtype == BF16 and y.shape == g.shape
        assert rel(y, want) <= tol + UBF
    # each matrix of the batch by itself: none is carried by the others' size
    worst = max(rel(a, b) for a, b in zip(y, want))
    assert worst <= 3 * tol + UBF


@pytest.mark.parametrize("kind", ["low rank", "exponential"])
@pytest.mark.parametrize("rows,cols", [(100, 90), (320, 640), (1024, 256)])
def test_other_spectra(rows, cols, kind):
    g = spectrum(kind, rows, cols, 2)
    want = iterate(g)
    assert rel(raw(g), want) <= tolerance(rows, cols, want / math.sqrt(2))
    assert rel(G.orthogonalize(g), want) <= tolerance(rows, cols, want / math.sqrt(2)) + UBF


def test_large_wide_batch():
    g = spectrum("strong directions", 1024, 4096, 3)
    assert rel(raw(g), iterate(g)) <= BLOCK
    t = g.transpose(1, 2).contiguous()
    assert rel(G.orthogonalize(t), iterate(t)) <= BLOCK + UBF


@pytest.mark.parametrize("steps,coefficients", [(1, G.NEWTON_SCHULZ), (2, G.NEWTON_SCHULZ), (7, G.NEWTON_SCHULZ), (12, (1.5, -0.5, 0.0)),
                                                (4, (G.NEWTON_SCHULZ, (3.4, -4.7, 2.0), (2.0, -1.5, 0.5), (1.875, -1.25, 0.375)))])
@pytest.mark.parametrize("rows,cols", [(96, 100), (300, 900)])
def test_steps_and_coefficients(rows, cols, steps, coefficients):
    g = torch.randn(2, rows, cols, device="cuda")
    want = iterate(g, steps, coefficients)
    # at most the growth of five of the usual steps in a block
    assert rel(raw(g, steps=steps, coefficients=coefficients), want) <= BLOCK
    assert rel(G.orthogonalize(g, steps=steps, coefficients=coefficients), want) <= BLOCK + UBF
    if steps == 12:      # the cubic iteration converges: rows orthonormal
        o = raw(g, steps=steps, coefficients=coefficients).double()
        smallest = torch.linalg.svdvals((g[0].double() / g[0].double().norm()).cpu())[-1].item()
        if smallest * 1.5 ** 9 > 1:
            assert (o[0] @ o[0].t() - torch.eye(rows, device="cuda", dtype=F64)).norm() / math.sqrt(rows) < 0.1


def test_size_of_the_gradient_does_not_matter():
    g = torch.randn(2, 150, 200, device="cuda")
    want = iterate(g)
    for scale in (2.0 ** 80, 2.0 ** -60, 1e30):
        assert rel(G.orthogonalize(g * scale, eps=0.0), want) <= tolerance(150, 200, want / math.sqrt(2)) + UBF + 2.0 ** -20
    tiny = iterate(g * 1e-9)     # eps counts here
    assert rel(G.orthogonalize(g * 1e-9), tiny) <= tolerance(150, 200, want / math.sqrt(2)) + UBF + 2.0 ** -20


def test_zero_and_not_finite_matrices_stay_by_themselves():
    for rows, cols in ((70, 50), (300, 400)):
        g = torch.randn(4, rows, cols, device="cuda")
        g[1] = 0
        g[2, 3, 4] = float("nan")
        g[3, 5, 6] = float("inf")
        y = G.orthogonalize(g)
        assert not y[1].any()
        assert torch.isnan(y[2]).any() and torch.isnan(y[3]).any()
        assert rel(y[0], iterate(g[0])) <= 3 * tolerance(rows, cols, iterate(g[0])) + UBF


def rounded(x, want, tol):
    """x, rounded to bf16 from something within tol of want, is as far from want as its rounding: rms of as many half steps as
    elements, equal for both but for four standard deviations of a mean square over them."""
    return rel(x, want) <= rel(want.to(BF16), want) * (1 + 4 / math.sqrt(want.numel())) + tol


@pytest.mark.parametrize("steps", [1, 5, 7])
@pytest.mark.parametrize("batch,rows,cols", [(2, 100, 120), (2, 120, 100), (70, 65, 130), (40, 200, 330), (9, 900, 400), (3, 1030, 2200), (2, 2200, 1030)])
def test_bf16_matrices(batch, rows, cols, steps):
    """bf16 matrices enter the first products unsplit: every tile, both orientations, one block and several."""
    x = spectrum("strong directions", rows, cols, batch).to(BF16)
    want = iterate(x, steps)
    assert rounded(G.orthogonalize(x, steps=steps), want, tolerance(rows, cols, want / math.sqrt(batch)))


@pytest.mark.parametrize("m", [1, 2, 32, 33, 64, 65, 96, 97, 128])
@pytest.mark.parametrize("n", [1, 5, 64, 100, 128, 129, 200, 255, 256, 257])
def test_small_matrices(m, n):
    """What one workgroup holds, and the first sizes beyond it: both orientations, both types, updates with momentum."""
    for rows, cols in ((m, n), (n, m)):
        g = spectrum("gaussian", rows, cols, 3)
        want = iterate(g)
        tol = tolerance(rows, cols, want / math.sqrt(3))
        got = raw(g)
        assert rel(got, want) <= tol and torch.equal(raw(g), got)
        for dtype in (F32, BF16):
            assert rel(G.orthogonalize(g.to(dtype)), iterate(g.to(dtype))) <= tol + UBF
        p, buf = torch.randn(3, rows, cols, device="cuda"), torch.randn(3, rows, cols, device="cuda")
        mom = 0.9 * buf.double() + 0.1 * g.double()
        u = 0.1 * g.double() + 0.9 * mom
        o = iterate(u)
        wantp = p.double() * (1 - 0.1 * 0.3) - 0.1 * 0.5 * o
        before = p.double().norm()
        G.muon_step(list(p), list(g), buf, lr=0.1, momentum=0.9, weight_decay=0.3, scale=0.5)
        # momentum: three fp32 operations on each element; parameters: the direction's tolerance and three operations
        assert (buf.double() - mom).norm() <= 4 * U32 * (buf.double().norm() + g.double().norm())
        assert (p.double() - wantp).norm() <= 0.05 * 2 * tol * o.norm() + 4 * U32 * (before + o.norm())


@pytest.mark.parametrize("m", [3, 40, 64, 70, 96, 100, 128])
@pytest.mark.parametrize("n", [300, 512, 1030, 4096, 4097])
def test_few_rows_in_strips(m, n):
    """A workgroup per 256 columns, and what has too many of them: both orientations and types, the same bits at every call."""
    for rows, cols in ((m, n), (n, m)):
        for batch in (2, 20):
            g = spectrum("gaussian", rows, cols, batch)
            want = iterate(g)
            tol = tolerance(rows, cols, want / math.sqrt(batch))
            got = raw(g)
            assert rel(got, want) <= tol and max(rel(a, b) for a, b in zip(got, want)) <= 3 * tol
            assert torch.equal(raw(g), got)
        x = g[:2].to(BF16)
        y = G.orthogonalize(x)
        assert rounded(y, iterate(x), tol)
        for _ in range(3):
            assert torch.equal(G.orthogonalize(x), y)


@pytest.mark.parametrize("rows,cols", [(150, 200), (700, 300)])
def test_bf16_matrices_of_any_size(rows, cols):
    g = spectrum("gaussian", rows, cols, 3).to(BF16)
    g[1] *= 3.0
    want = iterate(g)
    tol = tolerance(rows, cols, want / math.sqrt(3))
    for scale in (1.0, 2.0 ** 100, 2.0 ** -100, 1.7):
        x = g * scale
        assert rounded(G.orthogonalize(x, eps=0.0), want if scale != 1.7 else iterate(x), tol)
    x = g * 2.0 ** -30      # eps counts
    assert rounded(G.orthogonalize(x), iterate(x), tol)
    x = (g.double() * torch.exp(-24 * torch.rand(g.shape, device="cuda", dtype=F64))).to(BF16)     # elements of every size down to e^-24
    assert rounded(G.orthogonalize(x), iterate(x), tolerance(rows, cols, iterate(x) / math.sqrt(3)))


def test_bf16_zero_and_not_finite_matrices_stay_by_themselves():
    for rows, cols in ((70, 50), (300, 400)):
        g = torch.randn(6, rows, cols, device="cuda").to(BF16)
        g[1] = 0
        g[2, 3, 4] = float("nan")
        g[3, 5, 6] = float("inf")
        g[5] = 0
        for eps in (1e-7, 0.0):
            y = G.orthogonalize(g, eps=eps)
            assert not y[1].any() if eps else torch.isnan(y[1]).all()
            assert torch.isnan(y[2]).any() and torch.isnan(y[3]).any()
            for i in (0, 4):
                assert rel(y[i], iterate(g[i])) <= 3 * tolerance(rows, cols, iterate(g[i])) + UBF


def test_offsets_beyond_32_bits():
    store = torch.zeros((70, 8200, 8192), dtype=BF16, device="cuda")         # 4.7e9 elements
    for rows, cols in ((60, 50), (300, 40), (260, 8192)):
        g = store[:, 7900:7900 + rows, :cols]
        g.copy_(torch.randn(1, rows, cols, device="cuda"))
        g[-1] = torch.randn(rows, cols, device="cuda")
        y = G.orthogonalize(g)
        assert torch.equal(y[-1], G.orthogonalize(g[-1].contiguous())) and torch.equal(y[0], y[-2])
        out = store[:, :rows, :cols]
        assert torch.equal(G.orthogonalize(g.contiguous(), out=out), y)


def test_views_outputs_and_neighbours():
    base = torch.randn(5, 90, 140, device="cuda")
    for dtype in (F32, BF16):
        b = base.to(dtype)
        for v in (b[:, 3:80, 1:130], b[1::2, ::2, 4:100], b[2, :, :64], b[0], b[:, 7:8, :]):
            want = G.orthogonalize(v.contiguous())
            store = torch.full(v.shape[:-2] + (v.shape[-2] + 2, v.shape[-1] + 5), 9.0, dtype=BF16, device="cuda")
            out = store[..., 1:-1, 2:-3]
            assert torch.equal(G.orthogonalize(v, out=out), want) and torch.equal(out, want)
            store[..., 1:-1, 2:-3] = 9.0
            assert (store == 9.0).all()
            assert torch.equal(G.orthogonalize(v), want)       # the same bits again
    assert G.orthogonalize(torch.empty(0, 4, 5, device="cuda")).shape == (0, 4, 5)
    assert G.orthogonalize(torch.empty(3, 0, 5, device="cuda")).shape == (3, 0, 5)


def test_refusals():
    g = torch.randn(2, 8, 12, device="cuda")
    buf = torch.empty(2, 8, 12, dtype=BF16, device="cuda")
    for bad in (lambda: G.orthogonalize(g.half()), lambda: G.orthogonalize(g[0, 0]), lambda: G.orthogonalize(g.transpose(1, 2)),
                lambda: G.orthogonalize(g[:, :1].expand(2, 8, 12)), lambda: G.orthogonalize(g, out=buf[:1]), lambda: G.orthogonalize(g, out=g),
                lambda: G.orthogonalize(buf, out=buf), lambda: G.orthogonalize(g, steps=0), lambda: G.orthogonalize(g, steps=40),
                lambda: G.orthogonalize(g, coefficients=(30.0, 0.0, 0.0)),
                # singular values up to 1.3, 1.9, 12: the bound over their range grows, whatever these matrices hold
                lambda: G.orthogonalize(g, steps=4, coefficients=((4.0, -6.0, 3.0), (3.4, -4.7, 2.0), (2.5, -2.5, 1.0), (1.9, -1.3, 0.4))),
                lambda: G.orthogonalize(g, eps=-1.0),
                lambda: G.orthogonalize(g, out=torch.empty(8, 12, dtype=BF16, device="cuda").expand(2, 8, 12))):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    p, q, m = torch.randn(8, 12, device="cuda"), torch.randn(8, 12, device="cuda"), torch.zeros(8, 12, device="cuda")
    for params, grads, momenta in (([p], [q], [p]), ([p, p], [q, q], [m, torch.zeros_like(m)]), ([p], [p], [m]), ([p], [q.double()], [m]),
                                   ([p], [q[:, :11]], [m]), ([p], [q.t()], [m.t()]), ([p], [q], torch.zeros(2, 8, 12, device="cuda")),
                                   ([p], [m.view(-1)[:96].view(8, 12)], [m]), ([p], [q], [])):
        with pytest.raises(ValueError):
            G.muon_step(params, grads, momenta, 1e-3)


def reference_step(p, g, buf, lr, mu, nesterov, decay, scale):
    g = g.double()
    buf = mu * buf.double() + (1 - mu) * g
    u = (1 - mu) * g + mu * buf if nesterov else buf
    o = iterate(u)
    return (1 - lr * decay) * p.double() - lr * scale * o, buf, o


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("rows,cols,adjust", [(64, 64, "rms"), (33, 70, "spectral"), (300, 128, "spectral"), (768, 256, "rms"), (512, 1024, "rms")])
def test_optimizer_steps(rows, cols, adjust, nesterov):
    lr, mu, decay = 0.02, 0.9, 0.1
    params = [nn.Parameter(0.02 * torch.randn(rows, cols, device="cuda")) for _ in range(3)]
    idle = params[1].detach().clone()
    opt = training.Muon(params, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=decay, adjust=adjust)
    scale = 0.2 * math.sqrt(max(rows, cols)) if adjust == "rms" else math.sqrt(max(1, rows / cols))
    ref = {i: (params[i].detach().double(), torch.zeros(rows, cols, dtype=F64, device="cuda")) for i in (0, 2)}
    for step in range(3):
        for i in (0, 2):         # the middle one has no gradient
            params[i].grad = 1e-3 * spectrum("strong directions", rows, cols)[0]
        version = params[0]._version
        before = {i: params[i].detach().clone() for i in (0, 2)}
        opt.step()
        assert params[0]._version > version and torch.equal(params[1], idle) and not opt.momentum[0][1].any()
        for i in (0, 2):
            # from the parameters and momenta as they were, so that each step is judged by itself
            p, buf, o = reference_step(before[i], params[i].grad, ref[i][1].float(), lr, mu, nesterov, decay, scale)
            assert rel(opt.momentum[0][i], buf) <= 3 * 2.0 ** -24 + 2.0 ** -23
            off = (params[i].detach().double() - p).norm().item()
            # the direction's own rounding to fp32 before it is iterated counts as one more rounding of X
            assert off <= lr * scale * 1.1 * tolerance(rows, cols, o) * o.norm().item() + 4 * 2.0 ** -24 * p.norm().item()
            ref[i] = (p, opt.momentum[0][i].double())


def test_flat_parameters_and_adam_beside():
    named = [("m.encoder.layers.0.fc1.weight", nn.Parameter(torch.randn(64, 32, device="cuda"))),
             ("m.encoder.layers.0.fc1.bias", nn.Parameter(torch.randn(63, device="cuda"))),
             ("m.encoder.layers.1.fc1.weight", nn.Parameter(torch.randn(64, 32, device="cuda"))),
             ("m.projection.weight", nn.Parameter(torch.randn(16, 16, device="cuda")))]
    copies = [p.detach().clone() for _, p in named]
    flat = training.FlatParameters(named)
    matrices, rest = training.split_for_muon(named)
    opts = training.Muon(matrices, lr=0.01), training.Adam(rest, lr=0.01)
    flat.zero_grad()
    flat.grad.copy_(torch.randn(flat.total, device="cuda"))
    for o in opts:
        o.step()
    for (name, p), old in zip(named, copies):
        assert p.data_ptr() == flat.data.data_ptr() + 4 * flat.index[name][0]
        if ".encoder.layers." in name and p.dim() == 2:
            want, _, o = reference_step(old, p.grad, torch.zeros_like(old), 0.01, 0.95, True, 0.0, 0.2 * 8)
            assert (p.double() - want).norm() <= 0.016 * 1.1 * tolerance(64, 32, o) * o.norm() + 2.0 ** -22 * want.norm()
        else:
            assert not torch.equal(p, old)


def test_side_stream_and_replayed_graph():
    g = torch.randn(3, 100, 160, device="cuda")
    p, m = torch.randn(3, 100, 160, device="cuda"), torch.zeros(3, 100, 160, device="cuda")
    want = G.orthogonalize(g)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = G.orthogonalize(g)
    side.synchronize()
    assert torch.equal(got, want)
    p0, m0 = p.clone(), m.clone()

    def step(p, m):
        G.muon_step(list(p), list(g), m, 0.05)
        return G.orthogonalize(g)
    step(p0.clone(), m0.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step(p, m)
    p.copy_(p0)
    m.copy_(m0)
    for _ in range(4):
        g.copy_(torch.randn_like(g))
        graph.replay()
        torch.cuda.synchronize()
        e = step(p0, m0)
        torch.cuda.synchronize()
        assert torch.equal(o, e) and torch.equal(p, p0) and torch.equal(m, m0)


def test_fine_tuning_for_four_bits():
    """The operators as they are used together: a two-layer block fine-tuned through its 4-bit products with orthogonalised updates, the
    weights then quantised once and scored."""
    d, f, rows = 128, 256, 200
    w1, w2 = nn.Parameter(0.05 * torch.randn(f, d, device="cuda")), nn.Parameter(0.05 * torch.randn(d, f, device="cuda"))
    b1, b2 = nn.Parameter(torch.zeros(f, device="cuda")), nn.Parameter(torch.zeros(d, device="cuda"))
    opts = training.Muon([w1, w2], lr=0.02), training.Adam([b1, b2], lr=0.01)
    x = torch.randn(4, rows // 4, d, device="cuda").to(BF16)
    target = torch.randn(rows, d, device="cuda")

    def forward():
        u = training.linear_mxfp4(x, w1, b1)
        h = u * torch.sigmoid(1.702 * u)
        return training.linear_mxfp4(h, w2, b2), h
    for _ in range(3):
        for o in opts:
            o.zero_grad()
        y, h = forward()
        h.retain_grad()
        loss = (y.float().reshape(rows, d) - target).pow(2).mean()
        loss.backward()
        # the second layer's gradients are the formula's, on the quantised operands
        dy = (2 * (y.detach().float().reshape(rows, d) - target) / (rows * d)).to(BF16)
        dx, dw, db = G.linear_mxfp4_bwd(dy, ops.quantize_mxfp4(h.detach().reshape(rows, f)), ops.quantize_mxfp4(w2.detach()))
        # dy itself is formed by torch, in its own order of roundings: a bf16 step
        assert rel(w2.grad, dw.double()) <= 2 * UBF and rel(b2.grad, db.double()) <= 2 * UBF
        assert rel(h.grad.reshape(rows, f), dx.double()) <= 4 * UBF
        before = [p.detach().clone() for p in (w1, w2, b1, b2)]
        for o in opts:
            o.step()
        assert all(torch.isfinite(p).all() and not torch.equal(p, q) for p, q in zip((w1, w2, b1, b2), before))
    q1, q2 = ops.quantize_mxfp4(w1.detach()), ops.quantize_mxfp4(w2.detach())
    with torch.no_grad():
        u = training.linear_mxfp4(x, w1, b1).reshape(rows, f)
        assert torch.equal(ops.linear_mxfp4(x.reshape(rows, d), q1, b1.detach()), u)
        h = ops.linear_mxfp4(x.reshape(rows, d), q1, b1.detach(), gelu=True)
        res = torch.randn(rows, d, device="cuda")
        y = ops.linear_mxfp4(h, q2, b2.detach(), residual=res)
        assert torch.equal(training.linear_mxfp4(h, w2, b2), ops.linear_mxfp4(h, q2, b2.detach()))
        # the residual form adds before any rounding to bf16
        plain = ops.linear_mxfp4(h, q2, b2.detach(), residual=torch.zeros_like(res))
        assert ((y - (res + plain)).abs() <= 2.0 ** -22 * (res.abs() + plain.abs() + 1)).all()
