"""Linear products in 8-bit floating point (e4m3) with one scale for each block of 128, on sm_100a.

Activations are quantised by rows in blocks of 1 x 128, weights in blocks of 128 x 128:

    y[m, n] = sum_b sx[m, b] sw[n // 128, b] sum_{k in block b} q[m, k] w[n, k]  (+ bias[n])

Next to the W8A8 int8 linears this needs no Hadamard rotation (a block's outlier costs its own block
only) and has a gradient towards its input, for adapters trained through frozen quantised weights:
dx = quantised(dy) W, whose transposed weight has the same 128 x 128 blocks.
"""

from __future__ import annotations

import torch

from .. import _lib

BLOCK = 128


def fp8_block_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., K] (bf16, fp16, fp32) as e4m3 values [..., K] and fp32 scales [..., ceil(K / 128)].

    A block of 128 values with largest magnitude a has the scale 2^e, e >= -120 the least with
    a <= 448 * 2^e, so x / scale is exact and rounded once (to nearest, ties to even).  A block with an
    infinity or a NaN comes back NaN.  Rows of the values start on 16-byte boundaries.  Rounding has no
    gradient: the results are constants to autograd.
    """
    return _lib.ops().fp8_block_quantize(x)


def fp8_block_quantize_weight(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """w [N, K] (bf16, fp16, fp32) as e4m3 values [N, K] and fp32 scales [ceil(N/128), ceil(K/128)],
    one per block of 128 x 128, by the rule of ``fp8_block_quantize``."""
    return _lib.ops().fp8_block_quantize_weight(w)


def fp8_block_transpose(w_q: torch.Tensor) -> torch.Tensor:
    """w_q [N, K] of 8-bit values as [K, N] with 16-byte aligned rows (the scales transpose with it)."""
    return _lib.ops().fp8_block_transpose(w_q)


def fp8_block_matmul(x_q: torch.Tensor, x_scale: torch.Tensor, w_q: torch.Tensor, w_scale: torch.Tensor,
                     bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The product of quantised operands: x_q e4m3 [..., K], x_scale fp32 [..., ceil(K/128)], w_q e4m3
    [N, K], w_scale fp32 [ceil(N/128), ceil(K/128)] (any scales whose products stay within fp32's range,
    not only powers of two), bias of ``out_dtype`` [N] or None.  Sums in fp32, rounded once to ``out_dtype`` (bf16, fp16, fp32).  Not
    differentiable (its operands are not); ``fp8_block_linear`` is."""
    return _lib.ops().fp8_block_matmul(x_q, x_scale, w_q, w_scale, bias, out_dtype)


def fp8_block_linear(x: torch.Tensor, w_q: torch.Tensor, w_scale: torch.Tensor, bias: torch.Tensor | None = None,
                     w_q_t: torch.Tensor | None = None) -> torch.Tensor:
    """x [..., K] (bf16, fp16, fp32) through a block-quantised weight: [..., N] in x's type.

    x is quantised by rows in the call (``fp8_block_quantize``).  Differentiable once in x (dy is
    quantised by rows and multiplied with the transposed weight) and bias; the weight is a constant.
    ``w_q_t``: the weight laid out as [K, N] once by ``fp8_block_transpose``, for training; without it the
    backward pass transposes the weight in every call.  Weights whose rows do not start on 16-byte
    boundaries are copied in every call; ``fp8_block_quantize_weight`` and ``fp8_block_transpose`` lay
    them out so.
    """
    return _lib.ops().fp8_block_linear(x, w_q, w_scale, bias, w_q_t)


def _aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """t [R, C] of 8-bit values with rows on 16-byte boundaries, as the products read them: itself or a copy."""
    if t.stride(0) % 16 == 0 and t.stride(0) >= t.shape[1] and (t.stride(1) == 1 or t.shape[1] == 1):
        return t
    return t.new_zeros(t.shape[0], -(-t.shape[1] // 16) * 16)[:, :t.shape[1]].copy_(t)


class Fp8BlockLinear(torch.nn.Module):
    """A frozen linear layer on a block-quantised weight, differentiable in its input and bias.

    ``transposed=True`` keeps the weight laid out for the input's gradient too (another byte a weight).
    The weight's rows start on 16-byte boundaries, also after loading, casts and moves between devices, so
    that no call copies it; where a width is no multiple of 16 its buffers are views of padded rows.
    """

    def __init__(self, in_features: int, out_features: int, bias: bool = True, transposed: bool = False,
                 device=None, dtype=torch.bfloat16) -> None:
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        blocks = (-(-out_features // BLOCK), -(-in_features // BLOCK))
        kw = dict(device=device)
        zeros = lambda *shape: _aligned_rows(torch.zeros(*shape, dtype=torch.float8_e4m3fn, **kw))  # noqa: E731
        self.register_buffer("w_q", zeros(out_features, in_features))
        self.register_buffer("w_scale", torch.ones(blocks, dtype=torch.float32, **kw))
        self.register_buffer("w_q_t", zeros(in_features, out_features) if transposed else None)
        self.bias = torch.nn.Parameter(torch.zeros(out_features, dtype=dtype, **kw)) if bias else None

    @classmethod
    @torch.no_grad()
    def from_linear(cls, linear: torch.nn.Linear, transposed: bool = False) -> "Fp8BlockLinear":
        """The layer with ``linear``'s weight quantised (on its GPU) and its bias parameter, shared."""
        m = cls(linear.in_features, linear.out_features, bias=False, transposed=False, device="meta")
        m.w_q, m.w_scale = fp8_block_quantize_weight(linear.weight)
        m.w_q_t = fp8_block_transpose(m.w_q) if transposed else None
        m.bias = linear.bias
        return m

    def _apply(self, fn, recurse: bool = True):
        """``.to(dtype)``, ``.half()`` and the like change the bias alone: values and scales keep their types."""
        kept = {k: t for k, t in self._buffers.items() if t is not None}
        super()._apply(fn, recurse)
        for k, t in kept.items():
            if self._buffers[k].dtype != t.dtype:
                self._buffers[k] = t.to(self._buffers[k].device)
        self._lay_out()  # a move packs padded rows
        return self

    def _load_from_state_dict(self, *args, **kwargs):
        super()._load_from_state_dict(*args, **kwargs)
        self._lay_out()  # assign=True takes the loaded tensors as they are

    def _lay_out(self):
        for k in ("w_q", "w_q_t"):
            if self._buffers[k] is not None:
                self._buffers[k] = _aligned_rows(self._buffers[k])

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return fp8_block_linear(x, self.w_q, self.w_scale, self.bias, self.w_q_t)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, "
                f"transposed={self.w_q_t is not None}")
