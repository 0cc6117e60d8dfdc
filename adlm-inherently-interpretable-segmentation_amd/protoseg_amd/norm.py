"""Group norm with an activation on channels-last maps, forward and backward, on the HIP kernels.

    z = (x - mean) / sqrt(var + eps) * weight + bias        per (sample, group of channels)
    y = act(z),  act: identity, relu, sigmoid or silu

The reference's backbone normalises with BatchNorm and freezes it (segmentation/module.py:127),
because its micro-batch of 2 crops (cityscapes_kld_imnet.gin:23) is too small for batch
statistics; ``deeplab.DeepLabV2(norm="group")`` trains its normalisation at that batch with this
operator instead. Statistics are formed in f64, so a mean far larger than the spread costs no
accuracy, and all sums are joined in a fixed order (the same bits on every run).

A captured backward follows torch's rule for graphs: no eager autograd graph of the same leaves
may be alive while it is captured.
"""
from __future__ import annotations

import functools
from typing import Optional, Tuple

import torch
import torch.nn as nn
from torch import Tensor

from . import _lib
from .ops import _x_dtype

ACTIVATIONS = {"identity": 0, "relu": 1, "sigmoid": 2, "silu": 3}


def _rows(x: Tensor) -> Tuple[Tensor, int, int]:
    """x as the kernels read it, channel stride 1 and one stride from pixel to pixel, with its sample
    and pixel strides. A channels-last map, and a slice of one along batch or channels, passes as it
    is; anything else is copied. A stride that is never stepped over is given its dense value."""
    B, C, H, W = x.shape
    sb, sc, sh, sw = x.stride()
    sp = sw if W > 1 else sh if H > 1 else C
    if (sc == 1 or C == 1) and sp >= C and (H == 1 or W == 1 or sh == sw * W):
        if B == 1:
            return x, H * W * sp, sp
        if sb >= sp * (H * W - 1) + C:
            return x, sb, sp
    return x.contiguous(memory_format=torch.channels_last), H * W * C, C


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(code: int, B: int, HW: int, C: int, groups: int, backward: int) -> int:
    return _lib.load().protoseg_group_norm_workspace_size(code, B, HW, C, groups, backward)


def _empty_like_map(x: Tensor) -> Tensor:
    return torch.empty(x.shape, dtype=x.dtype, device=x.device, memory_format=torch.channels_last)


def _check(x: Tensor, groups: int, weight: Optional[Tensor], bias: Optional[Tensor], act: int) -> int:
    """Refuses what the kernels do not take; x's dtype code."""
    if x.dim() != 4:
        raise _lib.ProtosegError(f"group norm takes [B, C, H, W] maps; got {tuple(x.shape)}")
    code = _x_dtype(x)
    C = x.shape[1]
    if groups < 1 or C < 1 or C % groups:
        raise _lib.ProtosegError(f"{C} channels do not divide into {groups} groups")
    if weight is not None and (weight.dtype != torch.float32 or weight.shape != (C,)):
        raise _lib.ProtosegError(f"group norm weight: float32 [{C}] expected, got {weight.dtype} {tuple(weight.shape)}")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (C,)):
        raise _lib.ProtosegError(f"group norm bias: float32 [{C}] expected, got {bias.dtype} {tuple(bias.shape)}")
    if act not in ACTIVATIONS.values():
        raise _lib.ProtosegError(f"activation code {act} unknown")
    return code


def _forward(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], groups: int, eps: float, act: int):
    """y, stats and what a backward needs again: (x, weight, bias as read; the call's sizes)."""
    code = _check(x, groups, weight, bias, act)
    dev = _lib.require_device(x, weight, bias)
    x, sb, sp = _rows(x)
    weight = weight.contiguous() if weight is not None else None
    bias = bias.contiguous() if bias is not None else None
    B, C, H, W = x.shape
    y = _empty_like_map(x)
    stats = torch.empty((B, groups, 2), device=dev, dtype=torch.float64)
    sizes = (code, B, H * W, C, sb, sp)
    if x.numel() == 0:
        stats.zero_()
    else:
        lib = _lib.load()
        with _lib.on_device(dev):
            nbytes = _workspace_bytes(code, B, H * W, C, groups, 0)
            ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
            _lib.check("protoseg_group_norm_fwd", lib.protoseg_group_norm_fwd(
                x.data_ptr(), *sizes, groups, _lib.addr(weight), _lib.addr(bias), eps, act, y.data_ptr(), stats.data_ptr(),
                ws.data_ptr(), nbytes, _lib.stream_of(dev)))
    return y, stats, (x, weight, bias), sizes


def _backward(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], stats: Tensor, sizes, g_y: Tensor, groups: int,
              act: int, need_x: bool, need_weight: bool, need_bias: bool):
    """The backward on tensors that _forward returned; only g_y is new to it."""
    dev = x.device
    g_y, gsb, gsp = _rows(g_y if g_y.dtype == x.dtype else g_y.to(x.dtype))
    C = sizes[3]
    g_x = _empty_like_map(x) if need_x else None
    if x.numel() == 0:
        zero = x.new_zeros(C, dtype=torch.float32)
        return g_x, zero if need_weight else None, zero.clone() if need_bias else None
    g_w = torch.empty(C, device=dev, dtype=torch.float32) if need_weight else None
    g_b = torch.empty(C, device=dev, dtype=torch.float32) if need_bias else None
    lib = _lib.load()
    with _lib.on_device(dev):
        nbytes = _workspace_bytes(*sizes[:4], groups, 1)
        ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
        _lib.check("protoseg_group_norm_bwd", lib.protoseg_group_norm_bwd(
            x.data_ptr(), g_y.data_ptr(), *sizes, gsb, gsp, groups, _lib.addr(weight), _lib.addr(bias), act,
            stats.data_ptr(), _lib.addr(g_x), _lib.addr(g_w), _lib.addr(g_b), ws.data_ptr(), nbytes, _lib.stream_of(dev)))
    return g_x, g_w, g_b


def group_norm_forward(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], groups: int, eps: float,
                       act: int) -> Tuple[Tensor, Tensor]:
    """(y in x's dtype, channels last; f64 [B, groups, 2] means and reciprocal deviations). No autograd."""
    return _forward(x, weight, bias, groups, eps, act)[:2]


def group_norm_backward(x: Tensor, g_y: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], stats: Tensor, groups: int,
                        act: int, need_x: bool = True, need_weight: bool = True,
                        need_bias: bool = True) -> Tuple[Optional[Tensor], Optional[Tensor], Optional[Tensor]]:
    """Gradients of group_norm_forward's y with respect to (x, weight, bias); None where not needed."""
    code = _check(x, groups, weight, bias, act)
    _lib.require_device(x, g_y, weight, bias, stats)
    if g_y.shape != x.shape or stats.dtype != torch.float64 or tuple(stats.shape) != (x.shape[0], groups, 2):
        raise _lib.ProtosegError("group norm backward: g_y and stats must be of the forward's shapes")
    x, sb, sp = _rows(x)
    B, C, H, W = x.shape
    return _backward(x, weight.contiguous() if weight is not None else None, bias.contiguous() if bias is not None else None,
                     stats.contiguous(), (code, B, H * W, C, sb, sp), g_y, groups, act, need_x, need_weight, need_bias)


class _GroupNorm(torch.autograd.Function):
    # a Function and not a torch.library op as the layer's: its dispatch costs a training call more
    # host time than the kernels take on the backbone's maps at the micro-batch of 2
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        y, stats, used, ctx.sizes = _forward(x, weight, bias, groups, eps, act)
        ctx.save_for_backward(*used, stats)
        ctx.groups, ctx.act = groups, act
        return y

    @staticmethod
    def backward(ctx, g_y):
        if torch.is_grad_enabled():  # create_graph
            raise _lib.ProtosegError("group norm has no second derivative")
        return (*_backward(*ctx.saved_tensors, ctx.sizes, g_y, ctx.groups, ctx.act, *ctx.needs_input_grad[:3]), None, None, None)


def group_norm(x: Tensor, groups: int, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5,
               activation: str = "identity") -> Tensor:
    """Group norm of x [B, C, H, W] (float32, bfloat16 or float16) followed by ``activation``
    ("identity", "relu", "sigmoid" or "silu"): y of x's dtype, channels last.

    weight, bias: [C], float32 in the kernels (other floating types are widened, their gradients
    narrowed), or None. A channels-last x, and a slice of one along batch or channels, is read in
    place; any other layout is copied once. Gradients with respect to x, weight and bias.
    """
    if activation not in ACTIVATIONS:
        raise _lib.ProtosegError(f"activation {activation!r} has no HIP kernel (one of {sorted(ACTIVATIONS)})")
    if not eps >= 0:
        raise _lib.ProtosegError(f"group norm eps {eps}")
    if weight is not None and weight.dtype != torch.float32 and weight.is_floating_point():
        weight = weight.float()
    if bias is not None and bias.dtype != torch.float32 and bias.is_floating_point():
        bias = bias.float()
    args = (x, weight, bias, int(groups), float(eps), ACTIVATIONS[activation])
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _GroupNorm.apply(*args)
    return group_norm_forward(*args)[0]


class GroupNorm(nn.Module):
    """``group_norm`` with its affine parameters (torch.nn.GroupNorm's names), activation included."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, affine: bool = True,
                 activation: str = "identity"):
        super().__init__()
        if num_groups < 1 or num_channels < 1 or num_channels % num_groups:
            raise ValueError(f"{num_channels} channels do not divide into {num_groups} groups")
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation {activation!r} (one of {sorted(ACTIVATIONS)})")
        self.num_groups, self.num_channels, self.eps, self.activation = num_groups, num_channels, eps, activation
        self.affine = affine
        self.weight = nn.Parameter(torch.ones(num_channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(num_channels)) if affine else None

    def forward(self, x: Tensor) -> Tensor:
        return group_norm(x, self.num_groups, self.weight, self.bias, self.eps, self.activation)

    def extra_repr(self) -> str:
        return f"{self.num_groups}, {self.num_channels}, eps={self.eps}, affine={self.affine}, activation={self.activation}"
