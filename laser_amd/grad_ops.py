"""Torch-facing wrappers of the backward building blocks of libsgclip_hip.so.

Torch supplies device memory, the stream and views; every arithmetic step of the
train step's backward pass is one of the calls below (or `ops.gemm_bf16`).
"""
from __future__ import annotations

import ctypes as C
import functools
import os
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from .ops import Mxfp4, _apart, _ptr, _same_device, _stream, gemm_bf16

BF16, F32 = torch.bfloat16, torch.float32


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype == BF16:
        return _lib.DTYPE_BF16
    if t.dtype == F32:
        return _lib.DTYPE_F32
    raise TypeError(f"expected bf16 or f32, got {t.dtype}")


_TN_WGRAD = os.environ.get("SGCLIP_TN_WGRAD", "1") != "0"   # 0: transposed copies + the NT kernel (comparison)


def pad64(n: int) -> int:
    return (n + 63) // 64 * 64


def transpose_bf16(x: torch.Tensor, ld_out: Optional[int] = None) -> torch.Tensor:
    """bf16 [R, C] -> [C, ld_out] with out[c, r] = x[r, c]; columns R..ld_out-1 are zero."""
    assert x.dtype == BF16 and x.dim() == 2 and x.stride(1) == 1
    R, Cc = x.shape
    ld_out = ld_out or R
    out = torch.empty((Cc, ld_out), dtype=BF16, device=x.device)
    _lib.check(_lib.load().sgclip_transpose_bf16(x.data_ptr(), x.stride(0), R, Cc, out.data_ptr(), ld_out, _stream(x)))
    return out


def colsum(x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """f32 [N] (+)= column sums of x [M, N] (bf16 or f32)."""
    assert x.dim() == 2 and x.stride(1) == 1
    M, N = x.shape
    if out is None:
        out = torch.zeros(N, dtype=F32, device=x.device)
    _lib.check(_lib.load().sgclip_colsum(x.data_ptr(), _dtype_code(x), x.stride(0), M, N, out.data_ptr(), _stream(x)))
    return out


def quick_gelu(u: torch.Tensor) -> torch.Tensor:
    assert u.dtype == BF16 and u.is_contiguous()
    g = torch.empty_like(u)
    _lib.check(_lib.load().sgclip_quick_gelu(u.data_ptr(), g.data_ptr(), u.numel(), _stream(u)))
    return g


def quick_gelu_bwd(u: torch.Tensor, dg: torch.Tensor) -> torch.Tensor:
    assert u.dtype == BF16 and dg.dtype == BF16 and u.is_contiguous() and dg.is_contiguous() and u.shape == dg.shape
    du = torch.empty_like(u)
    _lib.check(_lib.load().sgclip_quick_gelu_bwd(u.data_ptr(), dg.data_ptr(), du.data_ptr(), u.numel(), _stream(u)))
    return du


def cast_bf16(x: torch.Tensor) -> torch.Tensor:
    assert x.dtype == F32 and x.is_contiguous()
    y = torch.empty(x.shape, dtype=BF16, device=x.device)
    _lib.check(_lib.load().sgclip_cast_f32_bf16(x.data_ptr(), y.data_ptr(), x.numel(), _stream(x)))
    return y


def cast_bf16_colsum(x: torch.Tensor, colsum_out: torch.Tensor) -> torch.Tensor:
    """bf16 copy of x (f32 [M, N]) with colsum_out (f32 [N]) += column sums of x, in one pass over x."""
    assert x.dtype == F32 and x.dim() == 2 and x.is_contiguous()
    M, N = x.shape
    if N % 8 or N > 2048:
        colsum(x, colsum_out)
        return cast_bf16(x)
    assert colsum_out.dtype == F32 and colsum_out.is_contiguous() and colsum_out.numel() == N
    y = torch.empty(x.shape, dtype=BF16, device=x.device)
    _lib.check(_lib.load().sgclip_cast_colsum_f32_bf16(x.data_ptr(), y.data_ptr(), M, N, colsum_out.data_ptr(), _stream(x)))
    return y


def fc2_dgrad_through_gelu(dy: torch.Tensor, w_t: torch.Tensor, u: torch.Tensor, zero_bias: torch.Tensor,
                           colsum_out: torch.Tensor) -> torch.Tensor:
    """du = (dy w_t^T) * quick_gelu'(u) (bf16 [M, N]) with colsum_out (f32 [N]) += column sums of du: the gradient at
    fc1's output and fc1's bias gradient from one GEMM (dy bf16 [M, K], w_t bf16 [N, K] = fc2's weight transposed)."""
    assert dy.dtype == BF16 and w_t.dtype == BF16 and u.dtype == BF16 and u.is_contiguous()
    assert dy.stride(1) == 1 and w_t.stride(1) == 1
    M, K = dy.shape
    N = w_t.shape[0]
    assert w_t.shape[1] == K and u.shape == (M, N)
    assert colsum_out.dtype == F32 and colsum_out.is_contiguous() and colsum_out.numel() == N and zero_bias.numel() >= N
    du = torch.empty_like(u)
    _lib.check(_lib.load().sgclip_gemm_mulgelugrad_bf16(dy.data_ptr(), dy.stride(0), w_t.data_ptr(), w_t.stride(0), du.data_ptr(),
                                                        N, M, N, K, zero_bias.data_ptr(), u.data_ptr(), colsum_out.data_ptr(),
                                                        _stream(dy)))
    return du


def layernorm_bwd(x: torch.Tensor, w: torch.Tensor, eps: float, dy: torch.Tensor, dw: torch.Tensor, db: torch.Tensor,
                  dx: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """dx (f32 [rows, d]; added to `dx` when accumulate) and dw / db (+=) of y = LayerNorm(x) w + b."""
    assert x.dtype == F32 and x.dim() == 2 and x.stride(1) == 1 and dy.is_contiguous() and dy.shape == x.shape
    rows, d = x.shape
    if dx is None:
        assert not accumulate
        dx = torch.empty((rows, d), dtype=F32, device=x.device)
    assert dx.dtype == F32 and dx.is_contiguous() and dx.shape == x.shape
    _lib.check(_lib.load().sgclip_layernorm_bwd(x.data_ptr(), x.stride(0), rows, d, w.data_ptr(), eps, dy.data_ptr(),
                                                _dtype_code(dy), dx.data_ptr(), 1 if accumulate else 0, dw.data_ptr(),
                                                db.data_ptr(), _stream(x)))
    return dx


def attention_bwd(qkv: torch.Tensor, dout: torch.Tensor, n_seq: int, T: int, heads: int, causal: bool,
                  key_mask: Optional[torch.Tensor] = None, dbias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """dqkv; with dbias (f32 [3d]) the column sums of dqkv are ADDED to it (the q | k | v bias gradient)."""
    assert qkv.dtype == BF16 and dout.dtype == BF16 and qkv.is_contiguous() and dout.is_contiguous()
    assert qkv.shape == (n_seq * T, 3 * heads * 64) and dout.shape == (n_seq * T, heads * 64)
    dqkv = torch.empty_like(qkv)
    if dbias is None:
        _lib.check(_lib.load().sgclip_attention_bwd(qkv.data_ptr(), dout.data_ptr(), dqkv.data_ptr(), n_seq, T, heads,
                                                    1 if causal else 0, _ptr(key_mask), _stream(qkv)))
    else:
        assert dbias.dtype == F32 and dbias.is_contiguous() and dbias.numel() == 3 * heads * 64
        _lib.check(_lib.load().sgclip_attention_bwd_bias(qkv.data_ptr(), dout.data_ptr(), dqkv.data_ptr(), dbias.data_ptr(), n_seq,
                                                         T, heads, 1 if causal else 0, _ptr(key_mask), _stream(qkv)))
    return dqkv


def matmul_f32(A: torch.Tensor, B: torch.Tensor, transA: bool = False, transB: bool = False, alpha: float = 1.0,
               out: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """alpha op(A) op(B) in fp32; A, B row-major 2-D."""
    assert A.dtype == F32 and B.dtype == F32 and A.stride(1) == 1 and B.stride(1) == 1
    M, K = (A.shape[1], A.shape[0]) if transA else A.shape
    Kb, N = (B.shape[1], B.shape[0]) if transB else B.shape
    assert K == Kb, (A.shape, B.shape, transA, transB)
    if out is None:
        assert not accumulate
        out = torch.empty((M, N), dtype=F32, device=A.device)
    _lib.check(_lib.load().sgclip_matmul_f32(A.data_ptr(), A.stride(0), 1 if transA else 0, B.data_ptr(), B.stride(0),
                                             1 if transB else 0, out.data_ptr(), out.stride(0), M, N, K, float(alpha),
                                             1 if accumulate else 0, _stream(A)))
    return out


def dot_f32(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """0-dim f32 <a, b>."""
    assert a.dtype == F32 and b.dtype == F32 and a.is_contiguous() and b.is_contiguous() and a.numel() == b.numel()
    out = torch.zeros((), dtype=F32, device=a.device)
    _lib.check(_lib.load().sgclip_dot_f32(a.data_ptr(), b.data_ptr(), a.numel(), out.data_ptr(), _stream(a)))
    return out


def prob_bwd(probs: torch.Tensor, dprobs: torch.Tensor, mode: int) -> torch.Tensor:
    assert probs.dtype == F32 and probs.is_contiguous() and dprobs.is_contiguous() and probs.shape == dprobs.shape
    K, N = probs.shape
    dl = torch.empty_like(probs)
    _lib.check(_lib.load().sgclip_prob_bwd(probs.data_ptr(), dprobs.data_ptr(), K, N, mode, dl.data_ptr(), _stream(probs)))
    return dl


def normalize_rows(x: torch.Tensor) -> torch.Tensor:
    assert x.dtype == F32 and x.is_contiguous() and x.dim() == 2
    y = torch.empty_like(x)
    _lib.check(_lib.load().sgclip_normalize_rows(x.data_ptr(), x.shape[0], x.shape[1], y.data_ptr(), _stream(x)))
    return y


def normalize_bwd(x: torch.Tensor, dxhat: torch.Tensor) -> torch.Tensor:
    assert x.dtype == F32 and x.is_contiguous() and dxhat.is_contiguous() and x.shape == dxhat.shape
    dx = torch.empty_like(x)
    _lib.check(_lib.load().sgclip_normalize_bwd(x.data_ptr(), dxhat.data_ptr(), x.shape[0], x.shape[1], dx.data_ptr(),
                                                _stream(x)))
    return dx


def segment_mean_bwd(dmean: torch.Tensor, seg: torch.Tensor, inv_count: torch.Tensor, N: int) -> torch.Tensor:
    assert dmean.dtype == F32 and dmean.is_contiguous() and seg.dtype == torch.int32 and inv_count.dtype == F32
    K, G = dmean.shape
    out = torch.empty((K, N), dtype=F32, device=dmean.device)
    _lib.check(_lib.load().sgclip_segment_mean_bwd(dmean.data_ptr(), seg.data_ptr(), inv_count.data_ptr(), K, N, G,
                                                   out.data_ptr(), _stream(dmean)))
    return out


def embed_text(table: torch.Tensor, pos: torch.Tensor, ids: torch.Tensor) -> torch.Tensor:
    """f32 [K*T, d] = table[ids] + pos[:T]; ids int32 [K, T] on the device."""
    assert table.dtype == F32 and pos.dtype == F32 and ids.dtype == torch.int32 and ids.is_contiguous()
    K, T = ids.shape
    d = table.shape[1]
    x = torch.empty((K * T, d), dtype=F32, device=table.device)
    _lib.check(_lib.load().sgclip_embed_text(table.data_ptr(), pos.data_ptr(), ids.data_ptr(), K, T, d, x.data_ptr(), _stream(table)))
    return x


def embed_cls(cls: torch.Tensor, pos: torch.Tensor, x: torch.Tensor, n_images: int, T: int):
    """Writes cls + pos[0] into row 0 of every image of x (f32 [n_images*T, d])."""
    d = x.shape[1]
    _lib.check(_lib.load().sgclip_embed_cls(cls.data_ptr(), pos.data_ptr(), n_images, T, d, x.data_ptr(), _stream(x)))


def rows_scatter_add(src: torch.Tensor, idx: torch.Tensor, dst: torch.Tensor):
    """dst[idx[r]] += src[r] (f32 rows)."""
    assert src.dtype == F32 and dst.dtype == F32 and src.is_contiguous() and dst.is_contiguous()
    assert idx.dtype == torch.int32 and idx.numel() == src.shape[0] and src.shape[1] == dst.shape[1]
    _lib.check(_lib.load().sgclip_rows_scatter_add(src.data_ptr(), idx.data_ptr(), src.shape[0], src.shape[1], dst.data_ptr(),
                                                   _stream(src)))


def adamw(param: torch.Tensor, grad: torch.Tensor, m: torch.Tensor, v: torch.Tensor, step: int, lr: float,
          beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8, weight_decay: float = 0.0):
    for t in (param, grad, m, v):
        assert t.dtype == F32 and t.is_contiguous() and t.numel() == param.numel()
    _lib.check(_lib.load().sgclip_adamw(param.data_ptr(), grad.data_ptr(), m.data_ptr(), v.data_ptr(), param.numel(), lr,
                                        beta1, beta2, eps, weight_decay, step, _stream(param)))


# -- linear layers on the MFMA GEMM ---------------------------------------------------------
def linear_dgrad(dy: torch.Tensor, w_t: torch.Tensor, zero_bias: torch.Tensor) -> torch.Tensor:
    """dx bf16 [M, in] = dy [M, out] W, with w_t = W^T stored [in, out] (bf16)."""
    M = dy.shape[0]
    dx = torch.empty((M, w_t.shape[0]), dtype=BF16, device=dy.device)
    return gemm_bf16(dy, w_t, dx, _lib.EPI_BIAS_BF16, bias=zero_bias)


def linear_wgrad(dy: torch.Tensor, x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out f32 [out, in] += dy^T x for dy bf16 [M, out], x bf16 [M, in] (out: zeros when omitted); M is zero-padded
    to a multiple of 64.  The reduction over M (all tokens of the batch) is split over workgroups that add into
    `out` atomically, so repeated calls accumulate."""
    M = dy.shape[0]
    if out is None:
        out = torch.zeros((dy.shape[1], x.shape[1]), dtype=F32, device=dy.device)
    assert out.dtype == F32 and out.shape == (dy.shape[1], x.shape[1]) and out.stride(1) == 1
    if _TN_WGRAD and dy.shape[1] % 8 == 0 and x.shape[1] % 8 == 0 and dy.stride(1) == 1 and x.stride(1) == 1 \
            and dy.stride(0) % 8 == 0 and x.stride(0) % 8 == 0 and dy.data_ptr() % 16 == 0 and x.data_ptr() % 16 == 0:
        # both operands as they lie in memory (rows = the reduction index); fragments are transposed on the LDS read
        _lib.check(_lib.load().sgclip_gemm_tn_bf16(dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), out.data_ptr(),
                                                   out.stride(0), dy.shape[1], x.shape[1], M, _stream(dy)))
        return out
    Mp = pad64(M)
    dyt = transpose_bf16(dy, Mp)
    xt = transpose_bf16(x, Mp)
    return gemm_bf16(dyt, xt, out, _lib.EPI_F32_ATOMIC)


# -- linear layers in 4-bit floats -----------------------------------------------------------
def column_sums(x: torch.Tensor) -> torch.Tensor:
    """f32 [N] column sums of x [M, N] (bf16 or f32), the same bits at every call (`colsum` adds with atomics, and to its output)."""
    if x.dim() != 2 or not x.is_cuda or (x.numel() and ((x.shape[1] > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < x.shape[1]))):
        raise ValueError(f"column_sums: expected [M, N] with contiguous rows on the GPU, got {tuple(x.shape)} {x.stride()} on {x.device}")
    M, N = x.shape
    lib = _lib.load()
    need = lib.sgclip_column_sums_workspace_bytes(M, N)
    out = torch.empty(N, dtype=F32, device=x.device)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    _lib.check(lib.sgclip_column_sums(x.data_ptr(), _dtype_code(x), x.stride(0) if M > 1 else max(N, 1), M, N, out.data_ptr(), _ptr(ws), need,
                                      _stream(x)))
    return out


def linear_mxfp4_bwd(dy: torch.Tensor, xq: Mxfp4, wq: Mxfp4, dx_dtype: torch.dtype = BF16, need_dx: bool = True, need_dw: bool = True,
                     need_db: bool = True) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(dx, dw, db) of y = xq wq^T + b for dy bf16 / f32 [M, N]: the gradient in the quantised operands, which a straight-through
    estimator hands to the unquantised ones.  dx [M, K] in dx_dtype, dw f32 [N, K], db f32 [N]; what is not needed is None.
    dy enters the products in bf16; the 4-bit operands enter exactly.  dw is summed with fp32 atomics (`linear_wgrad`)."""
    if dy.dim() != 2 or dy.dtype not in (BF16, F32) or dy.shape != (xq.rows, wq.rows) or xq.cols != wq.cols:
        raise ValueError(f"linear_mxfp4_bwd: dy {dy.dtype} {tuple(dy.shape)} for x {xq.shape} and weight {wq.shape}")
    if dx_dtype not in (BF16, F32):
        raise ValueError(f"linear_mxfp4_bwd: dx in {dx_dtype}")
    _same_device(dy, xq.data, wq.data)
    return linear_mxfp4_bwd_at(dy, (*xq.pointers(), *wq.pointers()), xq.rows, wq.rows, xq.cols, dx_dtype, need_dx, need_dw, need_db)


def linear_mxfp4_bwd_at(dy: torch.Tensor, operands, M: int, N: int, K: int, dx_dtype: torch.dtype, need_dx: bool, need_dw: bool, need_db: bool):
    """`linear_mxfp4_bwd`, unchecked, by the addresses of x's codes and scales and of the weight's (on dy's device)."""
    lib, dev = _lib.load(), dy.device
    if (N > 1 and dy.stride(1) != 1) or (M > 1 and dy.stride(0) < N):      # rows that are strided themselves, or overlap
        dy = dy.contiguous()
    dx = torch.empty((M, K), dtype=dx_dtype, device=dev) if need_dx else None
    dw = torch.empty((N, K), dtype=F32, device=dev) if need_dw else None
    db = torch.empty(N, dtype=F32, device=dev) if need_db else None
    head = (dy.data_ptr(), _dtype_code(dy), dy.stride(0) if M > 1 else N)
    need = lib.sgclip_mxfp4_linear_bwd_workspace_bytes(*head, M, N, K)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _lib.check(lib.sgclip_mxfp4_linear_bwd(*head, *operands, M, N, K, _ptr(dx), _lib.DTYPE_F32 if dx_dtype == F32 else _lib.DTYPE_BF16,
                                           _ptr(dw), _ptr(db), _ptr(ws), need, _stream(dy)))
    return dx, dw, db


# -- orthogonalised updates --------------------------------------------------------------------
NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)   # a, b, c: steepest at 0 with singular values kept within about 0.7 .. 1.2


@functools.lru_cache(maxsize=64)
def _coefficient_table(coefficients: tuple, steps: int):
    """C array f32 [steps][3] of one triple for all steps or of a triple per step."""
    rows = (coefficients,) * steps if not isinstance(coefficients[0], tuple) else coefficients
    if len(rows) != steps or any(len(r) != 3 for r in rows):
        raise ValueError(f"coefficients: one (a, b, c) or {steps} of them, got {coefficients}")
    return (C.c_float * (3 * steps))(*(float(v) for r in rows for v in r))


def _coefficients(coefficients, steps: int):
    if steps < 1:
        raise ValueError(f"{steps} Newton-Schulz steps")
    first = coefficients[0]
    key = tuple(tuple(float(v) for v in r) for r in coefficients) if isinstance(first, (tuple, list)) else tuple(float(v) for v in coefficients)
    return _coefficient_table(key, steps)


def orthogonalize(g: torch.Tensor, steps: int = 5, coefficients=NEWTON_SCHULZ, eps: float = 1e-7, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Newton-Schulz orthogonalisation of each matrix of g (bf16 / f32 [rows, cols] or [batch, rows, cols], rows contiguous):
    X = g / (|g| + eps), `steps` times X <- a X + (b A + c A^2) X with A = X X^T on the shorter side; bf16, shaped as g.
    coefficients: (a, b, c), or one such triple per step.  Operands of 22 bits and fp32 sums inside (off by 0.4 to 1.5 times
    what fp32 products are), one rounding at the end."""
    if g.dim() not in (2, 3) or g.dtype not in (BF16, F32) or g.device.type != "cuda":
        raise ValueError(f"orthogonalize: expected bf16 or f32 [rows, cols] or [batch, rows, cols] on the GPU, got {g.dtype} {tuple(g.shape)} on {g.device}")
    batch, (rows, cols) = (g.shape[0] if g.dim() == 3 else 1), g.shape[-2:]
    table = _coefficients(coefficients, steps)
    if out is None:
        out = torch.empty(g.shape, dtype=BF16, device=g.device)
    if out.shape != g.shape or out.dtype != BF16:
        raise ValueError(f"orthogonalize: out must be bf16 {tuple(g.shape)}, got {out.dtype} {tuple(out.shape)}")
    _same_device(g, out)
    if g.numel() == 0:
        return out
    for name, t in (("g", g), ("out", out)):
        if (cols > 1 and t.stride(-1) != 1) or (rows > 1 and t.stride(-2) < cols):
            raise ValueError(f"orthogonalize: rows of {name} must be contiguous and apart, got strides {t.stride()}")
    _apart("orthogonalize", out, g)
    ld = [t.stride(-2) if rows > 1 else cols for t in (g, out)]
    bs = [t.stride(0) if batch > 1 else rows * cols for t in (g, out)]
    lib = _lib.load()
    need = lib.sgclip_orthogonalize_workspace_bytes(batch, rows, cols)
    ws = torch.empty(need, dtype=torch.uint8, device=g.device)
    _lib.check(lib.sgclip_orthogonalize(g.data_ptr(), _dtype_code(g), bs[0], ld[0], batch, rows, cols, table, steps, eps, out.data_ptr(), bs[1],
                                        ld[1], ws.data_ptr(), need, _stream(g)))
    return out


def muon_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], momenta, lr: float, momentum: float = 0.95,
              nesterov: bool = True, weight_decay: float = 0.0, scale: float = 1.0, steps: int = 5, coefficients=NEWTON_SCHULZ,
              eps: float = 1e-7):
    """One orthogonalised-momentum step on matrices of one shape (contiguous f32 [rows, cols] each), in place:
    m = momentum m + (1 - momentum) g; u = (1 - momentum) g + momentum m (nesterov) or m;
    p = (1 - lr weight_decay) p - lr scale orthogonalize(u).  momenta: a list like the others, or one tensor [count, rows, cols].
    The matrices of a call share its launches."""
    n = len(params)
    if not n == len(grads) == len(momenta):
        raise ValueError(f"muon_step: {n} parameters, {len(grads)} gradients, {len(momenta)} momenta")
    if n == 0:
        return
    shape, dev = params[0].shape, params[0].device
    if len(shape) != 2 or dev.type != "cuda":
        raise ValueError(f"muon_step: expected matrices on the GPU, got {tuple(shape)} on {dev}")
    stacked = isinstance(momenta, torch.Tensor)
    for t in (*params, *grads, *((momenta,) if stacked else momenta)):
        if t.dtype != F32 or t.shape != ((n, *shape) if t is momenta else shape) or t.device != dev or not t.is_contiguous():
            raise ValueError(f"muon_step: every tensor must be contiguous f32 {tuple(shape)} on {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    size = 4 * shape[0] * shape[1]
    at = [[t.data_ptr() for t in params], [t.data_ptr() for t in grads],
          range(momenta.data_ptr(), momenta.data_ptr() + n * size, size) if stacked else [t.data_ptr() for t in momenta]]
    if size == 0:
        return
    # what is written must not lie in anything else that is read or written
    spans = sorted([(p, True) for p in at[0]] + [(p, False) for p in set(at[1])] + [(p, True) for p in at[2]])
    for (a, wa), (b, wb) in zip(spans, spans[1:]):
        if b < a + size and (wa or wb):
            raise ValueError("muon_step: parameters, gradients and momenta overlap, or one occurs twice")
    table = _coefficients(coefficients, steps)
    lib = _lib.load()
    tables = [(C.c_void_p * n)(*ps) for ps in at]
    need = lib.sgclip_orthogonalize_workspace_bytes(n, *shape)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _lib.check(lib.sgclip_muon_step(*tables, n, shape[0], shape[1], momentum, 1 if nesterov else 0, lr, weight_decay, scale, table, steps, eps,
                                    ws.data_ptr(), need, _stream(params[0])))
