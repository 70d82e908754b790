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
    beta_fast times are kept, a linear ramp between (Peng et al., arXiv 2309.00071).  The ramp runs over
    the number of turns, as in the paper's text; a ramp over the frequency's index gives other tables for
    the same parameters.  "original_length" may be given with any type; entries that a type does not
    have are refused.  Values are within a few steps of fp32 (2^-24 of each) of the exact ones, beside an
    error of the angle of 2^-55 turns for each unit of the position.
    """
    if isinstance(dim, bool) or not isinstance(dim, int) or dim < 2 or dim % 2:
        raise ValueError(f"dim must be a positive even number, got {dim!r}")
    kind, factor, original, fast, slow, attn = "none", 1.0, 0.0, 32.0, 1.0, 1.0
    if scaling:
        sc = dict(scaling)
        kind = sc.pop("type", None)
        if kind not in SCALINGS:
            raise ValueError(f"scaling type must be one of {tuple(SCALINGS)}, got {kind!r}")
        factor = float(sc.pop("factor", 1.0))
        if kind != "none" and not 1.0 <= factor < 1e9:
            raise ValueError(f"scaling factor must be at least 1, got {factor}")
        original = float(sc.pop("original_length", 0.0))
        if kind == "none" and factor != 1.0:
            raise ValueError(f"scaling type 'none' has no factor, got {factor}")
        if kind != "yarn" and sc:
            raise ValueError(f"scaling type {kind!r} has no entries {sorted(sc)}")
        fast, slow = float(sc.pop("beta_fast", 32.0)), float(sc.pop("beta_slow", 1.0))
        attn = sc.pop("attention_factor", None)
        if sc:
            raise ValueError(f"unknown scaling entries {sorted(sc)}")
        if kind == "yarn" and not (original > 0 and fast > slow):
            raise ValueError("yarn scaling needs original_length > 0 and beta_fast > beta_slow")
        attn = 0.1 * math.log(factor) + 1.0 if attn is None else float(attn)
        if not attn > 0:
            raise ValueError(f"attention_factor must be positive, got {attn}")
    T = 0
    if not isinstance(positions, torch.Tensor):
        positions, T = None, int(positions)
        if T < 0:
            raise ValueError(f"positions must not be negative, got {T}")
    return _lib.ops().rotary_table(positions, T, torch.device(device), dim, float(theta), SCALINGS[kind], factor,
                                   original, fast, slow, attn)


def rotary_embed(q: torch.Tensor, k: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor,
                 positions: torch.Tensor | None = None, layout: str = "interleaved"):
    """(q, k) with the first 2 * cos.shape[-1] features of every head turned; new contiguous tensors.

    q [B, S, H, D], k [B, S, Hk, D] or None, of one type (bf16, fp16, fp32), any strides; B <= 65535,
    D <= 1024.
    cos, sin: fp32 [L, R/2], or [B or 1, L, R/2]; row ``positions[b, s]`` turns token (b, s)
    (int32 or int64, broadcastable to [B, S]), row s where ``positions`` is None.  ``layout``:
    "interleaved" pairs features (2j, 2j+1), "half" pairs (j, j + R/2).  Features from R on pass
    through.  Tokens whose position lies outside the table come back NaN and set the device error
    word (``_lib.device_error_read_clear``).  Differentiable in q and k, any number of times.
    """
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}, got {layout!r}")
    return _lib.ops().rotary_embed(q, k, cos, sin, positions, layout == "half")
