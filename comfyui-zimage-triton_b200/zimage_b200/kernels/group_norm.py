"""Group normalisation with an activation on sm_100a, channels last, forward and backward."""

from __future__ import annotations

import functools
import math

import torch

from .. import _lib

ACTIVATIONS = {"none": 0, "silu": 1}
MAX_CHANNELS = 8192


@functools.lru_cache(maxsize=4096)
def _workspace(dev: int, B: int, P: int, C: int, G: int, backward: int) -> int:
    """Bytes of workspace on device ``dev`` (a function of the sizes alone), whole 16-byte pieces."""
    with torch.cuda.device(dev):
        return -(-_lib.load().zib_group_norm_workspace(B, P, C, G, backward) // 16) * 16


def _strides(x: torch.Tensor, P: int, C: int) -> tuple[torch.Tensor, int, int]:
    """x [B, ..., C] with its batch and position strides; a contiguous copy where it has no single one."""
    if x.is_contiguous():
        return x, P * C, C
    if x.dim() != 3:
        try:
            x = x.view(x.shape[0], P, C)
        except RuntimeError:
            x = x.contiguous()
            return x, P * C, C
    if x.stride(2) != 1 and C != 1:
        x = x.contiguous()
        return x, P * C, C
    return x, x.stride(0), x.stride(1)


def _forward(x, weight, bias, G, eps, act, P):
    """(y, buffer): y like x; the buffer starts with mean and 1/std, fp32 [B, G] each."""
    B, C = x.shape[0], x.shape[-1]
    dev = x.get_device()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = -(-8 * B * G // 16) * 16
    n = _workspace(dev, B, P, C, G, 0)
    buf = torch.empty(stats + n + 16, dtype=torch.uint8, device=x.device)
    at = buf.data_ptr()
    xs, sb, sp = _strides(x, P, C)
    wd = weight if weight is not None else bias
    _lib.call_on(dev, "zib_group_norm", xs.data_ptr(), sb, sp, y.data_ptr(),
                 None if weight is None else weight.data_ptr(), None if bias is None else bias.data_ptr(),
                 0 if wd is None else _lib.DTYPES[wd.dtype], at, at + 4 * B * G, at + stats, n, B, P, C, G,
                 _lib.DTYPES[x.dtype], eps, act)
    return y, buf


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, G, eps, act, P):
        y, buf = _forward(x, weight, bias, G, eps, act, P)
        ctx.save_for_backward(x, weight, bias, buf)
        ctx.conf = G, act, P
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise RuntimeError("group_norm_act is differentiable once: its gradient has no gradient of its own")
        x, weight, bias, buf = ctx.saved_tensors
        G, act, P = ctx.conf
        B, C = x.shape[0], x.shape[-1]
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        if x.numel() == 0:
            return (torch.empty_like(x) if want_x else None, torch.zeros_like(weight) if want_w else None,
                    torch.zeros_like(bias) if want_b else None, None, None, None, None)
        dev = x.get_device()
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if want_x else None
        dw = torch.empty_like(weight) if want_w else None
        db = torch.empty_like(bias) if want_b else None
        n = _workspace(dev, B, P, C, G, 1)
        ws = torch.empty(n, dtype=torch.uint8, device=x.device)
        xs, xsb, xsp = _strides(x, P, C)
        ds, dsb, dsp = _strides(dy, P, C)
        wd = weight if weight is not None else bias
        _lib.call_on(dev, "zib_group_norm_backward", xs.data_ptr(), xsb, xsp, ds.data_ptr(), dsb, dsp, _lib.ptr(dx),
                     _lib.ptr(weight), _lib.ptr(bias), 0 if wd is None else _lib.DTYPES[wd.dtype], _lib.ptr(dw),
                     _lib.ptr(db), buf.data_ptr(), buf.data_ptr() + 4 * B * G, ws.data_ptr(), n, B, P, C, G,
                     _lib.DTYPES[x.dtype], act)
        return dx, dw, db, None, None, None, None


def group_norm_act(x: torch.Tensor, num_groups: int, weight: torch.Tensor | None = None,
                   bias: torch.Tensor | None = None, eps: float = 1e-6, activation: str = "silu") -> torch.Tensor:
    """act((x - mean) / sqrt(var + eps) * weight + bias) over groups of the last dimension.

    x [B, ..., C] (bf16, fp16, fp32; channels last, any strides of the others); the mean and the
    variance of a batch entry's group run over its C / num_groups channels and every position
    between.  A convolution's [B, C, H, W] tensor in channels-last memory format is passed as
    ``x.permute(0, 2, 3, 1)`` without a copy.  weight, bias: [C] of one type (bf16, fp16, fp32),
    each may be None.  ``activation``: "silu" or "none".  Returns a contiguous tensor of x's shape
    and type; differentiable in x, weight and bias.
    """
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    shape = x.shape
    if len(shape) < 2:
        raise ValueError(f"x must be [B, ..., C], got {tuple(shape)}")
    C = shape[-1]
    if num_groups < 1 or C < 1 or C % num_groups:
        raise ValueError(f"{C} channels do not split into {num_groups} groups")
    if C > MAX_CHANNELS:
        raise RuntimeError(f"group_norm_act takes at most {MAX_CHANNELS} channels, got {C}")
    _lib.dtype_code(x, "x")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            if t.shape != (C,):
                raise ValueError(f"{name} must have shape ({C},), got {tuple(t.shape)}")
            _lib.dtype_code(t, name)
    if weight is not None and bias is not None and weight.dtype is not bias.dtype:
        raise ValueError(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    _lib.require_device(x)
    _lib.same_device(x, weight, bias)
    P = math.prod(shape[1:-1])
    if weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _GroupNorm.apply(x, weight, bias, num_groups, float(eps), act, P)
    return _forward(x, weight, bias, num_groups, float(eps), act, P)[0]


class GroupNormAct(torch.nn.Module):
    """``group_norm_act`` with its parameters; the names of ``torch.nn.GroupNorm``."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-6, affine: bool = True,
                 activation: str = "silu", device=None, dtype=None) -> None:
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
        if num_groups < 1 or num_channels % num_groups:
            raise ValueError(f"{num_channels} channels do not split into {num_groups} groups")
        self.num_groups, self.num_channels, self.eps, self.activation = num_groups, num_channels, eps, activation
        kw = dict(device=device, dtype=dtype)
        if affine:
            self.weight = torch.nn.Parameter(torch.ones(num_channels, **kw))
            self.bias = torch.nn.Parameter(torch.zeros(num_channels, **kw))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return group_norm_act(x, self.num_groups, self.weight, self.bias, self.eps, self.activation)

    def extra_repr(self) -> str:
        return f"{self.num_groups}, {self.num_channels}, eps={self.eps}, activation={self.activation}"
