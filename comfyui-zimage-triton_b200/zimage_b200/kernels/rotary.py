"""Rotary positions on sm_100a: queries and keys in one launch, and the cos/sin tables.

``triton_rope_3d`` rotates interleaved pairs of 128-wide bf16 heads by a complex table; the
operators here take any even head size, both pair layouts, a rotated part of the head, positions
gathered from a table, keys with fewer heads, three element types, and are differentiable (the
gradient of a rotation is the rotation by the opposite angle).
"""

from __future__ import annotations

import math

import torch

from .. import _lib

LAYOUTS = ("interleaved", "half")
SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}


def rotary_table(positions: torch.Tensor | int, dim: int, theta: float = 10000.0, scaling: dict | None = None,
                 device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin), fp32 [T, dim/2], of positions times theta^(-2j/dim).

    ``positions``: an int32 or int64 tensor [T] on the GPU, or a number T for 0 .. T-1 (on ``device``).
    ``scaling`` stretches the table over contexts longer than the trained one:
    {"type": "linear", "factor": f}, {"type": "ntk", "factor": f} (a larger base,
    theta f^(dim/(dim-2))) or {"type": "yarn", "factor": f, "original_length": n} with optional
    "beta_fast" (32), "beta_slow" (1) and "attention_factor" (0.1 ln f + 1): frequencies that turn
    less than beta_slow times over the original length are divided by f, those that turn more than
    beta_fast times are kept, a linear ramp between (Peng et al., arXiv 2309.00071).
    """
    if isinstance(dim, bool) or not isinstance(dim, int) or dim < 2 or dim % 2:
        raise ValueError(f"dim must be a positive even number, got {dim!r}")
    sc = dict(scaling or {"type": "none"})
    kind = sc.pop("type", None)
    if kind not in SCALINGS:
        raise ValueError(f"scaling type must be one of {tuple(SCALINGS)}, got {kind!r}")
    factor = float(sc.pop("factor", 1.0))
    if kind != "none" and not 1.0 <= factor < 1e9:
        raise ValueError(f"scaling factor must be at least 1, got {factor}")
    original = float(sc.pop("original_length", 0.0))
    fast, slow = float(sc.pop("beta_fast", 32.0)), float(sc.pop("beta_slow", 1.0))
    attn = sc.pop("attention_factor", None)
    if sc:
        raise ValueError(f"unknown scaling entries {sorted(sc)}")
    if kind == "yarn" and not (original > 0 and fast > slow):
        raise ValueError("yarn scaling needs original_length > 0 and beta_fast > beta_slow")
    attn = 0.1 * math.log(factor) + 1.0 if attn is None else float(attn)
    if not attn > 0:
        raise ValueError(f"attention_factor must be positive, got {attn}")
    if isinstance(positions, torch.Tensor):
        if positions.dim() != 1 or positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"positions must be an int32 or int64 vector, got {positions.dtype} "
                             f"{tuple(positions.shape)}")
        _lib.require_device(positions)
        T, dev, ptr = positions.shape[0], positions.device, positions.data_ptr()
        pos64, ps = int(positions.dtype == torch.int64), positions.stride(0)
    else:
        T, dev, ptr, pos64, ps = int(positions), torch.device(device), None, 0, 0
        if T < 0:
            raise ValueError(f"positions must not be negative, got {T}")
    cos = torch.empty(T, dim // 2, dtype=torch.float32, device=dev)
    sin = torch.empty(T, dim // 2, dtype=torch.float32, device=dev)
    _lib.call_on(_lib.require_device(cos), "zib_rotary_table", ptr, pos64, ps, 0, T, dim, float(theta), SCALINGS[kind], factor, original,
                 fast, slow, attn, cos.data_ptr(), sin.data_ptr())
    return cos, sin


def _rotate(q, k, cos, sin, positions, half: int, inverse: int):
    """One launch over q and k (either may be None): fresh contiguous outputs."""
    ref = q if q is not None else k
    B, S, _, D = ref.shape
    code, device = _lib.DTYPES[ref.dtype], ref.device
    args, outs, keep = [], [], []
    for t in (q, k):
        if t is None:
            args += (None, 0, 0, 0, None, 0)
            outs.append(None)
            continue
        sb, ss, sh, sd = t.stride()
        if (sd != 1 and D != 1) or (half == 0 and ((sb | ss | sh) & 1 or t.data_ptr() % (2 * t.element_size()))):
            t = t.contiguous()  # features side by side; interleaved, a pair is one access
            sb, ss, sh, sd = t.stride()
            keep.append(t)
        o = torch.empty(t.shape, dtype=t.dtype, device=device)
        args += (t.data_ptr(), sb, ss, sh, o.data_ptr(), t.shape[2])
        outs.append(o)
    if cos.dim() == 3:
        cs_b, cs_l, L = (0 if cos.shape[0] == 1 else cos.stride(0)), cos.stride(1), cos.shape[1]
    else:
        cs_b, cs_l, L = 0, cos.stride(0), cos.shape[0]
    if positions is None:
        pos = (None, 0, 0, 0)
    else:
        pos = (positions.data_ptr(), int(positions.dtype is torch.int64), *positions.stride())
    _lib.call_on(ref.get_device(), "zib_rotary", *args, code, cos.data_ptr(), sin.data_ptr(), cs_b, cs_l, L, *pos, B,
                 S, D, 2 * cos.shape[-1], half, inverse)
    return tuple(outs)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, half, inverse):
        ctx.save_for_backward(cos, sin, positions)
        ctx.conf = half, inverse
        ctx.set_materialize_grads(False)
        return _rotate(q, k, cos, sin, positions, half, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        if not ctx.needs_input_grad[0]:
            dq = None
        if not ctx.needs_input_grad[1]:
            dk = None
        gq = gk = None
        if dq is not None or dk is not None:
            cos, sin, positions = ctx.saved_tensors
            half, inverse = ctx.conf
            # the transposed map of a rotation is the rotation back, itself differentiable
            run = _Rotary.apply if torch.is_grad_enabled() else _rotate
            gq, gk = run(dq, dk, cos, sin, positions, half, 1 - inverse)
        return gq, gk, None, None, None, None, None


def rotary_embed(q: torch.Tensor, k: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor,
                 positions: torch.Tensor | None = None, layout: str = "interleaved"):
    """(q, k) with the first 2 * cos.shape[-1] features of every head turned; new contiguous tensors.

    q [B, S, H, D], k [B, S, Hk, D] or None, of one type (bf16, fp16, fp32), any strides.
    cos, sin: fp32 [L, R/2], or [B or 1, L, R/2]; row ``positions[b, s]`` turns token (b, s)
    (int32 or int64, broadcastable to [B, S]), row s where ``positions`` is None.  ``layout``:
    "interleaved" pairs features (2j, 2j+1), "half" pairs (j, j + R/2).  Features from R on pass
    through.  Tokens whose position lies outside the table come back NaN and set the device error
    word (``_lib.device_error_read_clear``).  Differentiable in q and k.
    """
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
    half = int(layout == "half")
    qs = q.shape
    if len(qs) != 4:
        raise ValueError(f"q must be [B, S, H, D], got {tuple(qs)}")
    B, S, _, D = qs
    dtype = q.dtype
    if k is not None:
        ks = k.shape
        if len(ks) != 4 or ks[0] != B or ks[1] != S or ks[3] != D or k.dtype is not dtype:
            raise ValueError(f"k {tuple(ks)} {k.dtype} does not go with q {tuple(qs)} {dtype}")
    cs = cos.shape
    if cs != sin.shape or len(cs) not in (2, 3) or cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
        raise ValueError(f"cos and sin must be fp32 tables of one shape, [L, R/2] or [B, L, R/2]; got "
                         f"{tuple(cs)} {cos.dtype} and {tuple(sin.shape)} {sin.dtype}")
    if len(cs) == 3 and cs[0] not in (1, B):
        raise ValueError(f"a table of {cs[0]} batch entries does not go with a batch of {B}")
    if not 1 <= cs[-1] <= D // 2:
        raise ValueError(f"tables of {cs[-1]} pairs do not go with heads of {D} features")
    if positions is None:
        if cs[-2] < S:
            raise ValueError(f"a table of {cs[-2]} rows is too short for {S} tokens")
    else:
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
        ps = positions.shape
        if len(ps) != 2 or ps[0] != B or ps[1] != S:
            try:
                positions = positions.expand(B, S)
            except RuntimeError:
                raise ValueError(f"positions {tuple(ps)} do not broadcast to {(B, S)}") from None
        if cs[-2] < 1:
            raise ValueError("empty table")
    _lib.dtype_code(q, "q")
    if not half and D % 2:
        raise ValueError(f"the interleaved layout needs an even head size, got {D}")
    if D > 1024:
        raise ValueError(f"heads of at most 1024 features, got {D}")
    _lib.require_device(q)
    _lib.same_device(q, k, cos, sin, positions)
    if cos.stride(-1) != 1 or cos.stride() != sin.stride():
        cos, sin = cos.contiguous(), sin.contiguous()
    if torch.is_grad_enabled():
        if cos.requires_grad or sin.requires_grad:
            raise ValueError("the tables of rotary_embed are constants: cos and sin must not require gradients")
        if q.requires_grad or (k is not None and k.requires_grad):
            return _Rotary.apply(q, k, cos, sin, positions, half, 0)
    return _rotate(q, k, cos, sin, positions, half, 0)
