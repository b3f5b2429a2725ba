"""Cases of the 4-bit linear layers and of the orthogonalised update, with their plain forms.

Five operators of the towers' linear layers:

  quantize  rows to microscaled 4-bit floats (e2m1 elements, one e8m0 scale per 32) and back to the values they stand for
  linear    epilogue(quantised x  times  quantised weight^T + bias), the form that scores
  train     the same product with its gradients, straight through the rounding
  ortho     Newton-Schulz orthogonalisation of a batch of matrices
  muon      one optimiser step with that orthogonalisation: momentum, direction, decay, update

A case holds plain values only.  `own` selects between the plain form (elementary torch operations in 32 or 64 bits) and the
framework's entry points.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 32
STEPS, COEFFS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
LR, MOMENTUM, DECAY = 1e-3, 0.95, 0.1
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}

# the largest listed case of each operator; drawn cases stay below
MOST = {"quantize": 73856 * 1024, "linear": 73856 * 1024 * 4096, "train": 36928 * 1024 * 4096, "ortho": 24 * 1024 * 1024 * 4096,
        "muon": 48 * 768 * 768 * 768}


def listed():
    return [
        # the token rows of one caption in the text tower: latency
        {"name": "quantize 77x512", "op": "quantize", "rows": 77, "cols": 512, "dtype": "bf16"},
        # the activations of 128 crops at 336 pixels (577 tokens each): bandwidth
        {"name": "quantize 73856x1024", "op": "quantize", "rows": 73856, "cols": 1024, "dtype": "bf16"},
        # one pooled token through the text tower's first MLP layer: latency of a single row
        {"name": "linear 1x512x2048", "op": "linear", "rows": 1, "k": 512, "n": 2048, "epilogue": "gelu", "dtype": "bf16"},
        # the pooled tokens of a few crops through a large tower's second MLP layer: the weights are the traffic
        {"name": "linear 7x4096x1024", "op": "linear", "rows": 7, "k": 4096, "n": 1024, "epilogue": "none", "dtype": "bf16"},
        # a vocabulary of 20 captions through the output projection of the large text tower, with the residual stream
        {"name": "linear 1540x768x768", "op": "linear", "rows": 1540, "k": 768, "n": 768, "epilogue": "residual", "dtype": "bf16"},
        # 128 crops at 336 pixels through the large image tower's first MLP layer: the matrix pipe and the output's bytes
        {"name": "linear 73856x1024x4096", "op": "linear", "rows": 73856, "k": 1024, "n": 4096, "epilogue": "gelu", "dtype": "bf16"},
        # fine-tuning on five captions: a small projection, forward and backward
        {"name": "train 385x512x512", "op": "train", "rows": 385, "k": 512, "n": 512},
        # fine-tuning on 64 crops at 336 pixels: the large tower's first MLP layer, forward and backward
        {"name": "train 36928x1024x4096", "op": "train", "rows": 36928, "k": 1024, "n": 4096},
        # two small matrices of odd sizes: launch latency and ragged tiles
        {"name": "ortho 2x127x255", "op": "ortho", "batch": 2, "rows": 127, "cols": 255, "dtype": "f32"},
        # the second MLP weights of all 24 layers of the large image tower
        {"name": "ortho 24x1024x4096", "op": "ortho", "batch": 24, "rows": 1024, "cols": 4096, "dtype": "bf16"},
        # the attention projections of the smallest geometry
        {"name": "muon 8x128x128", "op": "muon", "batch": 8, "rows": 128, "cols": 128},
        # the attention projections of all 12 layers of the base image tower
        {"name": "muon 48x768x768", "op": "muon", "batch": 48, "rows": 768, "cols": 768},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("quantize", "linear", "train", "ortho", "muon"))
    if op == "quantize":
        cols = _log_int(rng, 32, 4096)
        return {"op": op, "rows": _log_int(rng, 1, MOST[op] // cols), "cols": cols, "dtype": rng.choice(("bf16", "f32"))}
    if op == "linear":
        k, n = _log_int(rng, 64, 4096), _log_int(rng, 64, 4096)
        return {"op": op, "rows": _log_int(rng, 1, min(73856, MOST[op] // (k * n))), "k": k, "n": n,
                "epilogue": rng.choice(("none", "gelu", "residual")), "dtype": rng.choice(("bf16", "f32"))}
    if op == "train":
        k, n = _log_int(rng, 64, 4096), _log_int(rng, 64, 4096)
        return {"op": op, "rows": _log_int(rng, 1, min(36928, MOST[op] // (k * n))), "k": k, "n": n}
    a, b = _log_int(rng, 33, 2048 if op == "ortho" else 1024), _log_int(rng, 33, 2048 if op == "ortho" else 1024)
    case = {"op": op, "batch": _log_int(rng, 1, max(1, min(48, MOST[op] // (min(a, b) ** 2 * max(a, b))))), "rows": a, "cols": b}
    if op == "ortho":
        case["dtype"] = rng.choice(("bf16", "f32"))
    return case


def work(case):
    op = case["op"]
    if op == "quantize":
        n = case["rows"] * case["cols"]
        size = 2 if case["dtype"] == "bf16" else 4
        packed = case["rows"] * -(-case["cols"] // BLOCK) * 17
        return {"bytes": n * size + 2 * packed + n * 2, "flops": 0}
    if op == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        y = m * n * (8 if case["epilogue"] == "residual" else 2)
        return {"bytes": m * k * (2 if case["dtype"] == "bf16" else 4) + n * k * 17 // 32 + 4 * n + y, "flops": 2 * m * n * k}
    if op == "train":
        m, k, n = case["rows"], case["k"], case["n"]
        # x, weight, bias, y, dy read; the kept 4-bit operands written and read; dx, dw, db written
        return {"bytes": 2 * m * k + 4 * n * k + 4 * n + 4 * m * n + 2 * (m + n) * k * 17 // 32 + 2 * m * k + 4 * n * k + 4 * n,
                "flops": 6 * m * n * k}
    m, n, batch = min(case["rows"], case["cols"]), max(case["rows"], case["cols"]), case["batch"]
    # in terms of the Gram matrix: it and every polynomial of it are symmetric, half of each product is enough
    flops = batch * ((4 * STEPS - 3) * m ** 3 + 3 * m * m * n)
    if op == "ortho":
        return {"bytes": batch * m * n * ((2 if case["dtype"] == "bf16" else 4) + 2), "flops": flops}
    return {"bytes": batch * m * n * 20, "flops": flops}     # gradient read, momentum and parameters read and written


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(gen, rows, cols):
    """Layer-norm outputs as towers have them: normal values, every 50th channel or so ten times as large."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    loud = torch.rand(cols, generator=gen, device="cuda") < 0.02
    return x * (1 + 9 * loud.float())


def _gradients(gen, batch, rows, cols):
    """A few strong directions over a noise floor, the spectrum of a weight gradient."""
    rank = max(1, min(rows, cols) // 16)
    u = torch.randn(batch, rows, rank, generator=gen, device="cuda")
    v = torch.randn(batch, rank, cols, generator=gen, device="cuda")
    return 1e-3 * ((u @ v) / math.sqrt(rank) + 0.3 * torch.randn(batch, rows, cols, generator=gen, device="cuda"))


def _inputs(case, seed):
    gen, op = _generator(seed), case["op"]
    if op == "quantize":
        return {"x": _activations(gen, case["rows"], case["cols"]).to(DTYPES[case["dtype"]])}
    if op in ("linear", "train"):
        m, k, n = case["rows"], case["k"], case["n"]
        s = {"x": _activations(gen, m, k).to(DTYPES[case.get("dtype", "bf16")]),
             "w": 0.02 * torch.randn(n, k, generator=gen, device="cuda"),
             "b": 0.1 * torch.randn(n, generator=gen, device="cuda")}
        if case.get("epilogue") == "residual":
            s["r"] = torch.randn(m, n, generator=gen, device="cuda")
        if op == "train":
            s["dy"] = (1e-2 * torch.randn(m, n, generator=gen, device="cuda")).bfloat16()
        return s
    g = _gradients(gen, case["batch"], case["rows"], case["cols"])
    if op == "ortho":
        return {"g": g.to(DTYPES[case["dtype"]])}
    return {"g": g, "p": 0.02 * torch.randn(g.shape, generator=gen, device="cuda"),
            "buf": 0.5 * _gradients(gen, case["batch"], case["rows"], case["cols"])}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = dict(case)
    op = case["op"]
    if op == "linear":
        # a program that scores keeps its weights quantised: packed for the kernels, or as the values they stand for
        if own:
            from laser_amd import ops
            s["w"] = ops.quantize_mxfp4(s["w"])
        else:
            s["w"] = _as_mxfp4(s["w"])
    elif op == "train" and own:
        s["x"].requires_grad_(True)
        s["w"].requires_grad_(True)
        s["b"].requires_grad_(True)
    elif op == "muon" and own:
        from laser_amd import training
        params = [torch.nn.Parameter(p) for p in s["p"]]
        for p, g in zip(params, s["g"]):
            p.grad = g
        s["opt"] = training.Muon(params, lr=LR, momentum=MOMENTUM, weight_decay=DECAY)
        s["opt"].momentum[0].copy_(s["buf"])     # one stacked buffer per shape
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _as_mxfp4(x):
    """The values that x's microscaled 4-bit form stands for, in float32."""
    rows, cols = x.shape
    pad = -cols % BLOCK
    v = torch.nn.functional.pad(x.float(), (0, pad)).view(rows, -1, BLOCK)
    amax = v.abs().amax(-1, keepdim=True)
    e = (torch.frexp(amax)[1] - 3).clamp(-127, 127).double()
    e = torch.where(amax > 0, e, -127.0)
    y = v.abs().double() * torch.exp2(-e)        # 64 bits: next to a rounding border nothing may move
    q = 0.5 * ((y > 0.25).float() + (y >= 0.75) + (y > 1.25) + (y >= 1.75)) + (y > 2.5) + (y >= 3.5) + 2.0 * (y > 5.0)
    q = torch.where(v < 0, -q, q) * torch.exp2(e)
    q = torch.where(torch.isfinite(amax), q, math.nan)
    return q.float().view(rows, -1)[:, :cols]


def _quantize_plain(s):
    return _as_mxfp4(s["x"]).bfloat16()          # exact: bf16 holds every such value


def _linear_plain(s):
    y = _as_mxfp4(s["x"]) @ s["w"].t() + s["b"]
    epilogue = s["case"]["epilogue"]
    if epilogue == "residual":
        return s["r"] + y
    if epilogue == "gelu":
        y = y / (1 + torch.exp(-1.702 * y))
    return y.bfloat16()


def _train_plain(s):
    xq, wq, dy = _as_mxfp4(s["x"]), _as_mxfp4(s["w"]), s["dy"].float()
    y = xq @ wq.t() + s["b"]
    return {"y": y.bfloat16(), "dx": (dy @ wq).bfloat16(), "dw": dy.t() @ xq, "db": dy.sum(0)}


def _newton_schulz(u):
    """[batch, rows, cols] float32 -> the same, iterated on the shorter side."""
    flip = u.shape[1] > u.shape[2]
    x = u.transpose(1, 2).contiguous() if flip else u
    norm = x.double().square().sum((1, 2), keepdim=True).sqrt().float()
    x = x / (norm + EPS)
    a, b, c = COEFFS
    for _ in range(STEPS):
        gram = x @ x.transpose(1, 2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(1, 2) if flip else x


def _ortho_plain(s):
    return _newton_schulz(s["g"].float()).bfloat16().contiguous()


def _muon_plain(s):
    g, p, buf = s["g"], s["p"], s["buf"]
    buf.mul_(MOMENTUM).add_(g, alpha=1 - MOMENTUM)
    o = _newton_schulz((1 - MOMENTUM) * g + MOMENTUM * buf)
    scale = 0.2 * math.sqrt(max(p.shape[1:]))
    p.mul_(1 - LR * DECAY).add_(o, alpha=-LR * scale)
    return {"p": p, "momentum": buf}


def _quantize_own(s):
    from laser_amd import ops
    return ops.dequantize_mxfp4(ops.quantize_mxfp4(s["x"]))


def _linear_own(s):
    from laser_amd import ops
    epilogue = s["case"]["epilogue"]
    if epilogue == "residual":
        return ops.linear_mxfp4(s["x"], s["w"], s["b"], residual=s["r"])
    return ops.linear_mxfp4(s["x"], s["w"], s["b"], gelu=epilogue == "gelu")


def _train_own(s):
    from laser_amd import training
    y = training.linear_mxfp4(s["x"], s["w"], s["b"])
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def _ortho_own(s):
    from laser_amd import grad_ops
    return grad_ops.orthogonalize(s["g"], steps=STEPS, coefficients=COEFFS, eps=EPS)


def _muon_own(s):
    s["opt"].step()
    return {"p": s["p"], "momentum": s["opt"].momentum[0]}


_plain = {"quantize": _quantize_plain, "linear": _linear_plain, "train": _train_plain, "ortho": _ortho_plain, "muon": _muon_plain}
_own = {"quantize": _quantize_own, "linear": _linear_own, "train": _train_own, "ortho": _ortho_own, "muon": _muon_own}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _mxfp4_exact(x):
    """Written from the format: a shared exponent two below the block's largest, then round-half-even on the element's own step
    (1/2 below 2, 1 below 4, 2 from there), at most 6."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    v = torch.zeros(rows, blocks * BLOCK, dtype=torch.float64, device=x.device)
    v[:, :cols] = x
    v = v.view(rows, blocks, BLOCK)
    top = v.abs().max(dim=2, keepdim=True).values
    shared = torch.pow(2.0, torch.clamp(torch.floor(torch.log2(top)) - 2, min=-127, max=127))
    y = v / shared
    step = torch.full_like(y, 0.5)
    step[y.abs() >= 2] = 1.0
    step[y.abs() >= 4] = 2.0
    y = torch.clamp(torch.round(y / step) * step, -6, 6)
    return (y * shared).view(rows, -1)[:, :cols]


def _ortho_exact(u):
    """A step multiplies each singular value sigma by p(sigma^2), p(t) = a + b t + c t^2, and keeps the singular vectors.  So the
    result is the product of the steps' p(gram) times the first matrix, with gram -> p(gram) gram p(gram) between the steps."""
    flip = u.shape[1] > u.shape[2]
    x = (u.transpose(1, 2) if flip else u).double()
    x = x / (torch.linalg.vector_norm(x, dim=(1, 2), keepdim=True) + EPS)
    gram = torch.matmul(x, x.transpose(1, 2).contiguous())
    eye = torch.eye(x.shape[1], dtype=torch.float64, device=x.device)
    total = eye.expand_as(gram)
    for _ in range(STEPS):
        p = COEFFS[0] * eye + torch.matmul(gram, COEFFS[1] * eye + COEFFS[2] * gram)
        total = torch.matmul(p, total.contiguous())
        gram = torch.matmul(p, torch.matmul(gram, p))
    o = torch.matmul(total, x.contiguous())
    return o.transpose(1, 2).contiguous() if flip else o


def exact(case, seed):
    s, op = _inputs(case, seed), case["op"]
    if op == "quantize":
        return _mxfp4_exact(s["x"])
    if op in ("linear", "train"):
        xq, wq, b = _mxfp4_exact(s["x"]), _mxfp4_exact(s["w"]), s["b"].double()
        y = torch.addmm(b, xq, wq.t().contiguous())
        if op == "train":
            dy = s["dy"].double()
            return {"y": y, "dx": dy.mm(wq), "dw": dy.t().contiguous().mm(xq), "db": dy.sum(dim=0)}
        if case["epilogue"] == "gelu":
            return y * torch.sigmoid(1.702 * y)
        return y + s["r"].double() if case["epilogue"] == "residual" else y
    if op == "ortho":
        return _ortho_exact(s["g"])
    g = s["g"].double()
    buf = MOMENTUM * s["buf"].double() + (1 - MOMENTUM) * g
    u = (1 - MOMENTUM) * g + MOMENTUM * buf
    scale = 0.2 * math.sqrt(max(case["rows"], case["cols"]))
    return {"p": (1 - LR * DECAY) * s["p"].double() - LR * scale * _ortho_exact(u), "momentum": buf}
