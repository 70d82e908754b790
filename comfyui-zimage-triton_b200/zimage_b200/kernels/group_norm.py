"""Group normalisation with an activation on sm_100a, channels last, forward and backward."""

from __future__ import annotations

import torch

from .. import _lib

ACTIVATIONS = {"none": 0, "silu": 1}
MAX_CHANNELS = 8192


def _rows(x: torch.Tensor, B: int, P: int, C: int) -> torch.Tensor:
    """x as [B, P, C] with contiguous channels, a view where its strides allow one."""
    x3 = x.reshape(B, P, C)
    return x3 if x3.stride(2) == 1 or C == 1 else x3.contiguous()


def _forward(x3, groups, weight, bias, eps, act):
    B, P, C = x3.shape
    y = torch.empty(B, P, C, dtype=x3.dtype, device=x3.device)
    stats = torch.empty(2, B, groups, dtype=torch.float32, device=x3.device)
    wd = weight if weight is not None else bias
    ws = torch.empty(max(16, _workspace(x3, B, P, C, groups, 0)), dtype=torch.uint8, device=x3.device)
    _lib.call_on(x3, "zib_group_norm", x3.data_ptr(), x3.stride(0), x3.stride(1), y.data_ptr(), _lib.ptr(weight),
                 _lib.ptr(bias), 0 if wd is None else _lib.DTYPES[wd.dtype], stats[0].data_ptr(),
                 stats[1].data_ptr(), ws.data_ptr(), ws.numel(), B, P, C, groups, _lib.DTYPES[x3.dtype], eps, act)
    return y, stats


def _workspace(t, B, P, C, G, backward) -> int:
    lib = _lib.load()
    if t.get_device() == torch.cuda.current_device():
        return lib.zib_group_norm_workspace(B, P, C, G, backward)
    with torch.cuda.device(t.get_device()):
        return lib.zib_group_norm_workspace(B, P, C, G, backward)


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x3, weight, bias, groups, eps, act):
        y, stats = _forward(x3, groups, weight, bias, eps, act)
        ctx.save_for_backward(x3, weight, bias, stats)
        ctx.groups, ctx.act = groups, act
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x3, weight, bias, stats = ctx.saved_tensors
        B, P, C = x3.shape
        G = ctx.groups
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        if x3.numel() == 0:
            return (torch.empty_like(x3) if want_x else None, torch.zeros_like(weight) if want_w else None,
                    torch.zeros_like(bias) if want_b else None, None, None, None)
        if dy.stride(2) != 1 and C != 1:
            dy = dy.contiguous()
        dx = torch.empty(B, P, C, dtype=x3.dtype, device=x3.device) if want_x else None
        dw = torch.empty_like(weight) if want_w else None
        db = torch.empty_like(bias) if want_b else None
        wd = weight if weight is not None else bias
        ws = torch.empty(_workspace(x3, B, P, C, G, 1), dtype=torch.uint8, device=x3.device)
        _lib.call_on(x3, "zib_group_norm_backward", x3.data_ptr(), x3.stride(0), x3.stride(1), dy.data_ptr(),
                     dy.stride(0), dy.stride(1), _lib.ptr(dx), _lib.ptr(weight), _lib.ptr(bias),
                     0 if wd is None else _lib.DTYPES[wd.dtype], _lib.ptr(dw), _lib.ptr(db), stats[0].data_ptr(),
                     stats[1].data_ptr(), ws.data_ptr(), ws.numel(), B, P, C, G, _lib.DTYPES[x3.dtype], ctx.act)
        return dx, dw, db, None, None, None


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
    if x.dim() < 2:
        raise ValueError(f"x must be [B, ..., C], got {tuple(x.shape)}")
    B, C = x.shape[0], x.shape[-1]
    if num_groups < 1 or C < 1 or C % num_groups:
        raise ValueError(f"{C} channels do not split into {num_groups} groups")
    if C > MAX_CHANNELS:
        raise RuntimeError(f"group_norm_act takes at most {MAX_CHANNELS} channels, got {C}")
    _lib.dtype_code(x, "x")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.shape != (C,):
            raise ValueError(f"{name} must have shape ({C},), got {tuple(t.shape)}")
        if t is not None:
            _lib.dtype_code(t, name)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    _lib.require_device(x)
    _lib.same_device(x, weight=weight, bias=bias)
    P = 1
    for n in x.shape[1:-1]:
        P *= n
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    x3 = _rows(x, B, P, C)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        y = _GroupNorm.apply(x3, weight, bias, num_groups, float(eps), act)
    else:
        y = _forward(x3, num_groups, weight, bias, float(eps), act)[0]
    return y.view(x.shape)


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
