"""Group norm with an activation over channels-last images on MI355X.

New beside the reference, which optimizes its primitives directly: a network
that predicts them from an image, trained through the renderer, works on
channels-last images (the renderer's own layout) at batches of one or a few,
where group norm is the norm to use.  The norm, its scale and shift and the
activation are one operator with one backward; both run in
libcubicsplat_hip.so, in fp32 whatever the images' type.
"""
from __future__ import annotations

from functools import lru_cache
from typing import Optional

import torch

from . import _native as N
from . import torchcall

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "silu": 2, "gelu": 3}


def _channels_last(t: torch.Tensor) -> torch.Tensor:
    """t [N, C, ...] itself if its channels lie together and it has no gaps,
    else a copy that does."""
    if t.dim() == 4:
        return t if t.is_contiguous(memory_format=torch.channels_last) else \
            t.contiguous(memory_format=torch.channels_last)
    if t.dim() == 2:
        return t.contiguous()
    last = t.movedim(1, -1)
    return t if last.is_contiguous() else last.contiguous().movedim(-1, 1)


def _empty_channels_last(t: torch.Tensor) -> torch.Tensor:
    if t.dim() == 4:
        return torch.empty_like(t, memory_format=torch.channels_last)
    return torch.empty_like(t.movedim(1, -1), memory_format=torch.contiguous_format).movedim(-1, 1)


@lru_cache(maxsize=1024)
def _workspace_elems(n, s, c, groups, dtype, backward):
    return int(N.lib().cs_group_norm_workspace_elems(n, s, c, groups, dtype, backward))


def _param_ptr(p):
    return None if p is None else p.data_ptr()


def _forward(x, groups, weight, bias, eps, act):
    """y of x (channels last), and the mean and 1/deviation of each group
    ([2, N, groups] fp32)."""
    n, c = x.shape[0], x.shape[1]
    s = x.numel() // (n * c)
    y = _empty_channels_last(x)
    dtype = _DTYPES[x.dtype]
    work = torch.empty(_workspace_elems(n, s, c, groups, dtype, 0), dtype=torch.float32,
                       device=x.device)
    saved = torch.empty((2, n, groups), dtype=torch.float32, device=x.device)
    mean = saved.data_ptr()
    rstd = mean + 4 * n * groups
    affine = weight if weight is not None else bias
    with N.prof("norm.fwd"):
        N.call("cs_group_norm_forward", x.data_ptr(), n, s, c, groups, dtype, _param_ptr(weight),
               _param_ptr(bias), 0 if affine is None else _DTYPES[affine.dtype], eps, act,
               work.data_ptr(), mean, rstd, y.data_ptr(), N.stream(x.device))
    return y, saved


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        y, saved = _forward(x, groups, weight, bias, eps, act)
        ctx.save_for_backward(x, weight, bias, saved)
        ctx.groups, ctx.act = groups, act
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, saved = ctx.saved_tensors
        groups = ctx.groups
        n, c = x.shape[0], x.shape[1]
        s = x.numel() // (n * c)
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dy = _channels_last(dy)
        dtype = _DTYPES[x.dtype]
        dx = _empty_channels_last(x) if need_x else None
        dw = torch.empty_like(weight) if need_w else None
        db = torch.empty_like(bias) if need_b else None
        work = torch.empty(_workspace_elems(n, s, c, groups, dtype, 1), dtype=torch.float32,
                           device=x.device)
        affine = weight if weight is not None else bias
        mean = saved.data_ptr()
        with N.prof("norm.bwd"):
            N.call("cs_group_norm_backward", x.data_ptr(), dy.data_ptr(), n, s, c, groups, dtype,
                   _param_ptr(weight), _param_ptr(bias),
                   0 if affine is None else _DTYPES[affine.dtype], ctx.act, mean,
                   mean + 4 * n * groups, work.data_ptr(), _param_ptr(dx), _param_ptr(dw),
                   _param_ptr(db), N.stream(x.device))
        return dx, dw, db, None, None, None


def group_norm(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               activation: Optional[str] = None) -> torch.Tensor:
    """activation(torch.nn.functional.group_norm(x, num_groups, weight, bias, eps)).

    x: [N, C, ...] fp32, bf16 or fp16 on the GPU.  It is read where it lies if
    its memory is channels last without gaps ([N, ..., C], as
    ``torch.channels_last``) and copied to that layout otherwise; the result is
    channels last and of x's type.  weight and bias ([C], either may be absent)
    are of x's type or fp32.  activation: None, "relu", "silu" or "gelu" (erf).
    Mean, variance and everything that follows are computed in fp32 and rounded
    once.  Differentiable (once, in reverse mode; forward-mode derivatives are
    refused) in x, weight and bias; gradient sums are taken in a fixed order."""
    if x.dim() < 2:
        raise ValueError(f"expected [N, C, ...], got {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise ValueError(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    N.require_gpu(x, "x")
    c = x.shape[1]
    if num_groups < 1 or c < 1 or c % num_groups:
        raise ValueError(f"{c} channels cannot be divided into {num_groups} groups")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be None, 'relu', 'silu' or 'gelu', got {activation!r}")
    if not eps >= 0.0:
        raise ValueError(f"Invalid eps: {eps}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.shape != (c,):
            raise ValueError(f"{name} must have shape ({c},), got {tuple(p.shape)}")
        if p.dtype is not x.dtype and p.dtype is not torch.float32:
            raise ValueError(f"{name} must be {x.dtype} or float32, got {p.dtype}")
        if p.device != x.device:
            raise ValueError(f"{name} is on {p.device}, x on {x.device}")
    if weight is not None and bias is not None and weight.dtype is not bias.dtype:
        raise ValueError(f"weight and bias differ in type: {weight.dtype} and {bias.dtype}")
    if x.numel() == 0:
        return x * 1.0 if weight is None and bias is None else _empty(x, weight, bias)
    if weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if x.device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(x.device):
            return group_norm(x, num_groups, weight, bias, eps, activation)
    x = _channels_last(x)
    act = _ACTIVATIONS[activation]
    ext = torchcall.module()
    if ext is not None and N._PROFILE_CTX_FACTORY is None:
        return ext.group_norm(x, weight, bias, int(num_groups), float(eps), act)
    # Without the extension, or where each launch is bracketed by a context manager.
    return _GroupNorm.apply(x, weight, bias, int(num_groups), float(eps), act)


def _empty(x, weight, bias):
    """An empty result that hands zero gradients to the parameters."""
    shape = (1, x.shape[1]) + (1,) * (x.dim() - 2)
    y = x
    if weight is not None:
        y = y * weight.view(shape).to(x.dtype)
    if bias is not None:
        y = y + bias.view(shape).to(x.dtype)
    return y


class GroupNorm(torch.nn.GroupNorm):
    """torch.nn.GroupNorm (its parameters and state_dict) followed by an
    activation, as group_norm computes both."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, affine: bool = True,
                 device=None, dtype=None, *, activation: Optional[str] = None):
        super().__init__(num_groups, num_channels, eps, affine, device=device, dtype=dtype)
        if activation not in _ACTIVATIONS:
            raise ValueError(
                f"activation must be None, 'relu', 'silu' or 'gelu', got {activation!r}")
        self.activation = activation

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return group_norm(x, self.num_groups, self.weight, self.bias, self.eps, self.activation)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, activation={self.activation}"
