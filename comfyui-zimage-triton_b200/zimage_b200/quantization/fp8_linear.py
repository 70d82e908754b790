"""Linear products in 8-bit floating point (e4m3) with one scale for each block of 128, on sm_100a.

Activations are quantised by rows in blocks of 1 x 128, weights in blocks of 128 x 128:

    y[m, n] = sum_b sx[m, b] sw[n // 128, b] sum_{k in block b} q[m, k] w[n, k]  (+ bias[n])

Next to the W8A8 int8 linears this needs no Hadamard rotation (a block's outlier costs its own block
only) and has a gradient towards its input, for adapters trained through frozen quantised weights:
dx = quantised(dy) W, whose transposed weight has the same 128 x 128 blocks.
"""

from __future__ import annotations

import functools

import torch

from .. import _lib

BLOCK = 128
E4M3 = torch.float8_e4m3fn


def _empty_rows(rows: int, cols: int, device) -> torch.Tensor:
    """e4m3 [rows, cols] whose rows start on 16-byte boundaries."""
    ld = -(-cols // 16) * 16
    t = torch.empty(rows, ld, dtype=E4M3, device=device)
    return t if ld == cols else t[:, :cols]


def _rows(x: torch.Tensor, K: int) -> torch.Tensor:
    """x [..., K] as [M, K] with contiguous columns and rows that do not overlap."""
    x2 = x.reshape(-1, K)
    return x2 if x2.stride(1) == 1 and (x2.stride(0) >= K or x2.shape[0] <= 1) else x2.contiguous()


def _ld(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1])


def _aligned(q: torch.Tensor) -> torch.Tensor:
    """8-bit [R, C] with contiguous columns and 16-byte aligned rows: q itself, or a copy."""
    if (q.stride(1) == 1 or q.shape[1] == 1) and q.data_ptr() % 16 == 0 and \
            (q.shape[0] <= 1 or (q.stride(0) % 16 == 0 and q.stride(0) >= q.shape[1])):
        return q
    t = _empty_rows(q.shape[0], q.shape[1], q.device)
    t.copy_(q)
    return t


def _ld16(t: torch.Tensor) -> int:
    return -(-t.shape[1] // 16) * 16 if t.shape[0] <= 1 else t.stride(0)


def _quant_rows(x2: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(q [M, K], s [ceil(K/128), M]) of rows x2."""
    M, K = x2.shape
    q = _empty_rows(M, K, x2.device)
    s = torch.empty(-(-K // BLOCK), M, dtype=torch.float32, device=x2.device)
    _lib.call_on(x2.get_device(), "zib_fp8_quant_rows", x2.data_ptr(), _ld(x2), _lib.DTYPES[x2.dtype],
                 q.data_ptr(), _ld16(q), s.data_ptr(), 1, M, M, K)
    return q, s


def fp8_block_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., K] (bf16, fp16, fp32) as e4m3 values [..., K] and fp32 scales [..., ceil(K / 128)].

    A block of 128 values with largest magnitude a has the scale 2^e, e >= -120 the least with
    a <= 448 * 2^e, so x / scale is exact and rounded once (to nearest, ties to even).  A block with an
    infinity or a NaN comes back NaN.  Rows of the values start on 16-byte boundaries.
    """
    _lib.dtype_code(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be [..., K] with K >= 1, got {tuple(x.shape)}")
    _lib.require_device(x)
    lead, K = x.shape[:-1], x.shape[-1]
    q, s = _quant_rows(_rows(x.detach(), K))
    s = s.t()
    if len(lead) == 1:
        return q, s
    return (q.unflatten(0, lead), s.unflatten(0, lead)) if lead else (q[0], s[0])


def fp8_block_quantize_weight(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """w [N, K] (bf16, fp16, fp32) as e4m3 values [N, K] and fp32 scales [ceil(N/128), ceil(K/128)],
    one per block of 128 x 128, by the rule of ``fp8_block_quantize``."""
    _lib.dtype_code(w, "w")
    if w.dim() != 2 or w.numel() == 0:
        raise ValueError(f"w must be a non-empty [N, K], got {tuple(w.shape)}")
    _lib.require_device(w)
    w = _rows(w.detach(), w.shape[1])
    N, K = w.shape
    q = _empty_rows(N, K, w.device)
    s = torch.empty(-(-N // BLOCK), -(-K // BLOCK), dtype=torch.float32, device=w.device)
    _lib.call_on(w.get_device(), "zib_fp8_quant_blocks", w.data_ptr(), _ld(w), _lib.DTYPES[w.dtype],
                 q.data_ptr(), _ld16(q), s.data_ptr(), s.stride(0), 1, N, K)
    return q, s


def fp8_block_transpose(w_q: torch.Tensor) -> torch.Tensor:
    """w_q [N, K] of 8-bit values as [K, N] with 16-byte aligned rows (the scales transpose with it)."""
    if w_q.dim() != 2 or w_q.dtype != E4M3 or w_q.numel() == 0:
        raise ValueError(f"w_q must be a non-empty e4m3 [N, K], got {w_q.dtype} {tuple(w_q.shape)}")
    _lib.require_device(w_q)
    if w_q.stride(1) != 1 or w_q.stride(0) < w_q.shape[1]:
        w_q = w_q.contiguous()
    N, K = w_q.shape
    t = _empty_rows(K, N, w_q.device)
    _lib.call_on(w_q.get_device(), "zib_fp8_transpose", w_q.data_ptr(), _ld(w_q), t.data_ptr(), _ld16(t), N, K)
    return t


def _check_weight(K: int, w_q, w_scale, bias, dtype) -> int:
    """Refuses what does not go together; returns N."""
    shape = w_q.shape
    if len(shape) != 2 or w_q.dtype is not E4M3 or shape[1] != K or shape[0] < 1:
        raise ValueError(f"w_q must be e4m3 [N, {K}], got {w_q.dtype} {tuple(shape)}")
    N = shape[0]
    if w_scale.shape != (-(-N // BLOCK), -(-K // BLOCK)) or w_scale.dtype is not torch.float32:
        raise ValueError(f"w_scale must be fp32 {(-(-N // BLOCK), -(-K // BLOCK))}, got {w_scale.dtype} "
                         f"{tuple(w_scale.shape)}")
    if bias is not None and (bias.shape != (N,) or bias.dtype is not dtype):
        raise ValueError(f"bias must be {dtype} ({N},), got {bias.dtype} {tuple(bias.shape)}")
    return N


def fp8_block_matmul(x_q: torch.Tensor, x_scale: torch.Tensor, w_q: torch.Tensor, w_scale: torch.Tensor,
                     bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The product of quantised operands: x_q e4m3 [..., K], x_scale fp32 [..., ceil(K/128)], w_q e4m3
    [N, K], w_scale fp32 [ceil(N/128), ceil(K/128)] (any scales, not only powers of two), bias of
    ``out_dtype`` [N] or None.  Sums in fp32, rounded once to ``out_dtype`` (bf16, fp16, fp32)."""
    if x_q.dim() < 1 or x_q.dtype != E4M3 or x_q.shape[-1] < 1:
        raise ValueError(f"x_q must be e4m3 [..., K], got {x_q.dtype} {tuple(x_q.shape)}")
    K = x_q.shape[-1]
    if x_scale.shape != (*x_q.shape[:-1], -(-K // BLOCK)) or x_scale.dtype != torch.float32:
        raise ValueError(f"x_scale must be fp32 {(*x_q.shape[:-1], -(-K // BLOCK))}, got {x_scale.dtype} "
                         f"{tuple(x_scale.shape)}")
    if out_dtype not in _lib.DTYPES:
        raise ValueError(f"out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
    _check_weight(K, w_q, w_scale, bias, out_dtype)
    _lib.require_device(x_q)
    _lib.same_device(x_q, x_scale, w_q, w_scale, bias)
    sx = x_scale.reshape(-1, x_scale.shape[-1])
    q, w = _aligned(x_q.reshape(-1, K)), _aligned(w_q)
    bias = None if bias is None else bias.contiguous()
    M, N = q.shape[0], w.shape[0]
    y = torch.empty(*x_q.shape[:-1], N, dtype=out_dtype, device=q.device)
    _lib.call_on(q.get_device(), "zib_fp8_block_gemm", q.data_ptr(), _ld16(q), sx.data_ptr(), sx.stride(0),
                 sx.stride(1), w.data_ptr(), _ld16(w), w_scale.data_ptr(), w_scale.stride(0), w_scale.stride(1),
                 _lib.ptr(bias), y.data_ptr(), N, _lib.DTYPES[out_dtype], M, N, K)
    return y


@functools.lru_cache(maxsize=4096)
def _scratch_bytes(M: int, K: int, with_sum: int) -> int:
    return _lib.load().zib_fp8_block_linear_scratch(M, K, with_sum)


def _linear(x, w, sw, sw_n, sw_k, bias, shape, col_sum=None):
    """x [..., K] (rows as ``_lead_rows`` leaves them) through w [N, K]: a fresh tensor of ``shape``;
    the sums of x's columns into ``col_sum``."""
    N, K = w.shape
    M = x.numel() // K
    device = x.device
    y = torch.empty(shape, dtype=x.dtype, device=device)
    n = _scratch_bytes(M, K, col_sum is not None)
    scratch = torch.empty(n, dtype=torch.uint8, device=device) if n else None
    _lib.call_on(x.get_device(), "zib_fp8_block_linear", x.data_ptr(), K if x.is_contiguous() else x.stride(0),
                 _lib.DTYPES[x.dtype], w.data_ptr(), _ld16(w), sw.data_ptr(), sw_n, sw_k,
                 None if bias is None else bias.data_ptr(), y.data_ptr(), N,
                 None if col_sum is None else col_sum.data_ptr(), None if scratch is None else scratch.data_ptr(), n,
                 M, N, K)
    return y


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, bias, w_q, w_scale, w_q_t, shape):
        ctx.save_for_backward(w_q, w_scale, w_q_t)
        ctx.shape = x.shape
        return _linear(x, w_q, w_scale, w_scale.stride(0), w_scale.stride(1), bias, shape)

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise RuntimeError("fp8_block_linear is differentiable once: its gradient has no gradient of its own")
        w_q, w_scale, w_q_t = ctx.saved_tensors
        N = w_q.shape[0]
        dy = _lead_rows(dy, N)
        dx = db = None
        if ctx.needs_input_grad[1]:
            db = torch.empty(N, dtype=dy.dtype, device=dy.device)
        if ctx.needs_input_grad[0]:  # the pass that quantises dy adds up its columns too
            wt = _aligned(w_q_t) if w_q_t is not None else fp8_block_transpose(w_q)
            dx = _linear(dy, wt, w_scale, w_scale.stride(1), w_scale.stride(0), None, ctx.shape, db)
        elif db is not None:
            ws = torch.empty(64 * N, dtype=torch.float32, device=dy.device)
            _lib.call_on(dy.get_device(), "zib_col_sum", dy.data_ptr(), N if dy.is_contiguous() else dy.stride(0),
                         _lib.DTYPES[dy.dtype], db.data_ptr(), ws.data_ptr(), ws.numel() * 4, dy.numel() // N, N)
        return dx, db, None, None, None, None


def _lead_rows(x: torch.Tensor, K: int) -> torch.Tensor:
    """x [..., K] itself where its rows are a fixed step apart (contiguous, or a matrix with contiguous
    columns), else a contiguous copy."""
    if x.is_contiguous() or (x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= K):
        return x
    return x.contiguous()


def fp8_block_linear(x: torch.Tensor, w_q: torch.Tensor, w_scale: torch.Tensor, bias: torch.Tensor | None = None,
                     w_q_t: torch.Tensor | None = None) -> torch.Tensor:
    """x [..., K] (bf16, fp16, fp32) through a block-quantised weight: [..., N] in x's type.

    x is quantised by rows in the call (``fp8_block_quantize``).  Differentiable in x (dy is quantised
    by rows and multiplied with the transposed weight) and bias; the weight is a constant.  ``w_q_t``:
    the weight laid out as [K, N] once by ``fp8_block_transpose``, for training; without it the backward
    pass transposes the weight in every call.
    """
    dtype = x.dtype
    _lib.dtype_code(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be [..., K] with K >= 1, got {tuple(x.shape)}")
    K = x.shape[-1]
    N = _check_weight(K, w_q, w_scale, bias, dtype)
    if w_q_t is not None and (w_q_t.shape != (K, N) or w_q_t.dtype != E4M3):
        raise ValueError(f"w_q_t must be e4m3 ({K}, {N}), got {w_q_t.dtype} {tuple(w_q_t.shape)}")
    _lib.require_device(x)
    _lib.same_device(x, w_q, w_scale, bias, w_q_t)
    grad = torch.is_grad_enabled()
    if grad and (w_scale.requires_grad or w_q.requires_grad):
        raise ValueError("the quantised weight of fp8_block_linear is a constant and must not require gradients")
    w = _aligned(w_q)
    shape = (*x.shape[:-1], N)
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if grad and (x.requires_grad or (bias is not None and bias.requires_grad)):
        return _Linear.apply(_lead_rows(x, K), bias, w, w_scale, w_q_t, shape)
    return _linear(_lead_rows(x, K), w, w_scale, w_scale.stride(0), w_scale.stride(1), bias, shape)
