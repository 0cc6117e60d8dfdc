"""Group norm with an activation on channels-last maps, forward and backward, on the HIP kernels.

    z = (x - mean) / sqrt(var + eps) * weight + bias        per (sample, group of channels)
    y = act(z),  act: identity, relu, sigmoid or silu

The reference's backbone normalises with BatchNorm and freezes it (segmentation/module.py:127),
because its micro-batch of 2 crops (cityscapes_kld_imnet.gin:23) is too small for batch
statistics; ``deeplab.DeepLabV2(norm="group")`` trains its normalisation at that batch with this
operator instead. Statistics are sums in f64 of differences to a value of the group itself, so a mean
far larger than the spread (2^20 spreads in float32) costs no accuracy, and all sums are joined in a
fixed order (the same bits on every run).

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

ACTIVATIONS = {"identity": 0, "relu": 1, "sigmoid": 2, "silu": 3}


# Beside its kernels a training call on the backbone's maps is host time, most of it Python objects that the
# autograd thread and the caller's take from each other's caches. So what types, shapes and strides decide is
# worked out once for each of them, and a call looks it up.
@functools.lru_cache(maxsize=4096)
def _strides(shape: torch.Size, stride: Tuple[int, ...]) -> Optional[Tuple[int, int]]:
    """Sample and pixel stride of a map as the kernels read it, channel stride 1 and one stride from pixel to
    pixel: a channels-last map, and a slice of one along batch or channels. None: anything else, which is
    copied. A stride that is never stepped over is given its dense value."""
    B, C, H, W = shape
    sb, sc, sh, sw = stride
    sp = sw if W > 1 else sh if H > 1 else C
    if (sc == 1 or C == 1) and sp >= C and (H == 1 or W == 1 or sh == sw * W):
        if B == 1:
            return H * W * sp, sp
        if sb >= sp * (H * W - 1) + C:
            return sb, sp
    return None


def _rows(x: Tensor) -> Tuple[Tensor, int, int]:
    """x, or its channels-last copy, and its strides."""
    at = _strides(x.shape, x.stride())
    if at is not None:
        return (x, *at)
    B, C, H, W = x.shape
    return x.contiguous(memory_format=torch.channels_last), H * W * C, C


_CODES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


@functools.lru_cache(maxsize=4096)
def _sizes(dtype: torch.dtype, shape: torch.Size, groups: int) -> Tuple[Tuple[int, int, int, int], int, int]:
    """(dtype code, B, HW, C) and the workspace bytes of a forward and of a backward. Refuses what the kernels do
    not take."""
    if len(shape) != 4:
        raise _lib.ProtosegError(f"group norm takes [B, C, H, W] maps; got {tuple(shape)}")
    if dtype not in _CODES:
        raise _lib.ProtosegError(f"feature map dtype {dtype} unsupported (float32, bfloat16 or float16)")
    B, C, H, W = shape
    if groups < 1 or C < 1 or C % groups:
        raise _lib.ProtosegError(f"{C} channels do not divide into {groups} groups")
    sizes = (_CODES[dtype], B, H * W, C)
    if B > 65535 or H * W > 1 << 30 or C > 1 << 20:
        raise _lib.ProtosegError(f"group norm of {B} maps of {H * W} pixels and {C} channels (at most 65535, 2^30 and 2^20)")
    nbytes = _lib.load().protoseg_group_norm_workspace_size
    return sizes, nbytes(*sizes, groups, 0), nbytes(*sizes, groups, 1)


def _check_affine(name: str, t: Optional[Tensor], C: int, index: int) -> Optional[Tensor]:
    if t is None:
        return None
    if t.dtype != torch.float32 or t.shape != (C,):
        raise _lib.ProtosegError(f"group norm {name}: float32 [{C}] expected, got {t.dtype} {tuple(t.shape)}")
    if t.get_device() != index:
        raise _lib.ProtosegError(f"group norm {name} on {t.device}: the map's device expected")
    return t.contiguous()


def _forward(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], groups: int, eps: float, act: int):
    """y, stats and what a backward needs again: (x, weight, bias) as read, and the call's sizes and x's layout."""
    plan = _sizes(x.dtype, x.shape, groups)
    sizes, nbytes = plan[0], plan[1]
    if not 0 <= act < len(ACTIVATIONS):
        raise _lib.ProtosegError(f"activation code {act} unknown")
    index = x.get_device()
    weight, bias = _check_affine("weight", weight, sizes[3], index), _check_affine("bias", bias, sizes[3], index)
    if index < 0:
        _lib.require_device(x)  # refuses
    x, *at = _rows(x)
    y = torch.empty_like(x, memory_format=torch.channels_last)
    stats = x.new_empty((sizes[1], groups, 2), dtype=torch.float64)
    if sizes[1] == 0 or sizes[2] == 0:
        stats.zero_()
    else:
        ws = x.new_empty(nbytes, dtype=torch.uint8)
        _lib.call_on(index, "protoseg_group_norm_fwd", x.data_ptr(), *sizes, *at, groups, _lib.addr(weight),
                     _lib.addr(bias), eps, act, y.data_ptr(), stats.data_ptr(), ws.data_ptr(), nbytes)
    return y, stats, (x, weight, bias), (plan, x.stride(), at)


def _backward(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], stats: Tensor, plan, g_y: Tensor, groups: int,
              act: int, need_x: bool, need_weight: bool, need_bias: bool):
    """The backward on the values that _forward returned. Hooks on saved tensors (a map kept in host memory meanwhile)
    may have given them another layout."""
    (sizes, _, nbytes), stride, at = plan
    if x.stride() != stride:
        x, *at = _rows(x)
    weight, bias = weight if weight is None else weight.contiguous(), bias if bias is None else bias.contiguous()
    C = sizes[3]
    g_x = torch.empty_like(x, memory_format=torch.channels_last) if need_x else None
    if sizes[1] == 0 or sizes[2] == 0:
        zero = x.new_zeros(C, dtype=torch.float32)
        return g_x, zero if need_weight else None, zero.clone() if need_bias else None
    g_y, *g_at = _rows(g_y if g_y.dtype == x.dtype else g_y.to(x.dtype))
    g_w = x.new_empty(C, dtype=torch.float32) if need_weight else None
    g_b = x.new_empty(C, dtype=torch.float32) if need_bias else None
    stats = stats.contiguous()
    ws = x.new_empty(nbytes, dtype=torch.uint8)
    _lib.call_on(x.get_device(), "protoseg_group_norm_bwd", x.data_ptr(), g_y.data_ptr(), *sizes, *at, *g_at, groups,
                 _lib.addr(weight), _lib.addr(bias), act, stats.data_ptr(), _lib.addr(g_x), _lib.addr(g_w), _lib.addr(g_b),
                 ws.data_ptr(), nbytes)
    return g_x, g_w, g_b


def group_norm_forward(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], groups: int, eps: float,
                       act: int) -> Tuple[Tensor, Tensor]:
    """(y in x's dtype, channels last; f64 [B, groups, 2] means and reciprocal deviations). No autograd."""
    if not _lib.direct(x, weight, bias):
        with torch.no_grad():
            return torch.ops.protoseg.group_norm(x, weight, bias, groups, eps, act)
    return _forward(x, weight, bias, groups, eps, act)[:2]


def group_norm_backward(x: Tensor, g_y: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], stats: Tensor, groups: int,
                        act: int, need_x: bool = True, need_weight: bool = True,
                        need_bias: bool = True) -> Tuple[Optional[Tensor], Optional[Tensor], Optional[Tensor]]:
    """Gradients of group_norm_forward's y with respect to (x, weight, bias); None where not needed."""
    need = need_x, need_weight, need_bias
    if not _lib.direct(x, g_y, weight, bias, stats):
        with torch.no_grad():
            grads = torch.ops.protoseg.group_norm_backward(x, g_y, weight, bias, stats, groups, act, *need)
        return tuple(g if n else None for g, n in zip(grads, need))
    return _checked_backward(x, g_y, weight, bias, stats, groups, act, *need)


def _checked_backward(x, g_y, weight, bias, stats, groups, act, need_x, need_weight, need_bias):
    plan = _sizes(x.dtype, x.shape, groups)
    C = plan[0][3]
    if not 0 <= act < len(ACTIVATIONS):
        raise _lib.ProtosegError(f"activation code {act} unknown")
    _lib.require_device(x, g_y, weight, bias, stats)
    if g_y.shape != x.shape or stats.dtype != torch.float64 or tuple(stats.shape) != (x.shape[0], groups, 2):
        raise _lib.ProtosegError("group norm backward: g_y and stats must be of the forward's shapes")
    weight, bias = _check_affine("weight", weight, C, x.get_device()), _check_affine("bias", bias, C, x.get_device())
    return _backward(x, weight, bias, stats, (plan, None, None), g_y, groups, act, need_x, need_weight, need_bias)


# The operators for tracers, compilers and dispatch modes. Other calls do without: an operator's dispatch costs a
# training call more host time than the kernels take on the backbone's maps at the micro-batch of 2.
@torch.library.custom_op("protoseg::group_norm", mutates_args=(), device_types="cuda")
def _group_norm_op(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], groups: int, eps: float,
                   act: int) -> Tuple[Tensor, Tensor]:
    """group_norm_forward."""
    return _forward(x, weight, bias, groups, eps, act)[:2]


@_group_norm_op.register_fake
def _(x, weight, bias, groups, eps, act):
    return (torch.empty_like(x, memory_format=torch.channels_last),
            x.new_empty((x.shape[0], groups, 2), dtype=torch.float64))


@torch.library.custom_op("protoseg::group_norm_backward", mutates_args=(), device_types="cuda")
def _group_norm_backward_op(x: Tensor, g_y: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], stats: Tensor, groups: int,
                            act: int, need_x: bool, need_weight: bool, need_bias: bool) -> Tuple[Tensor, Tensor, Tensor]:
    """group_norm_backward; gradients that are not needed are empty."""
    grads = _checked_backward(x, g_y, weight, bias, stats, groups, act, need_x, need_weight, need_bias)
    none = (x.dtype, torch.float32, torch.float32)
    return tuple(x.new_empty(0, dtype=dt) if g is None else g for g, dt in zip(grads, none))


@_group_norm_backward_op.register_fake
def _(x, g_y, weight, bias, stats, groups, act, need_x, need_weight, need_bias):
    C = x.shape[1]
    return (torch.empty_like(x, memory_format=torch.channels_last) if need_x else x.new_empty(0),
            x.new_empty(C if need_weight else 0, dtype=torch.float32), x.new_empty(C if need_bias else 0, dtype=torch.float32))


def _op_setup(ctx, inputs, output):
    x, weight, bias, groups, _, act = inputs
    ctx.save_for_backward(x, weight, bias, output[1])
    ctx.call = groups, act
    ctx.mark_non_differentiable(output[1])


def _op_backward(ctx, g_y, _):
    x, weight, bias, stats = ctx.saved_tensors
    need = ctx.needs_input_grad[:3]
    grads = torch.ops.protoseg.group_norm_backward(x, g_y, weight, bias, stats, *ctx.call, *need)
    return (*(g if n else None for g, n in zip(grads, need)), None, None, None)


_group_norm_op.register_autograd(_op_backward, setup_context=_op_setup)


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        y, stats, used, plan = _forward(x, weight, bias, groups, eps, act)
        ctx.save_for_backward(*used, stats)
        ctx.call = plan, groups, act
        return y

    @staticmethod
    def backward(ctx, g_y):
        if torch.is_grad_enabled():  # create_graph
            raise _lib.ProtosegError("group norm has no second derivative")
        plan, groups, act = ctx.call
        need = ctx.needs_input_grad
        return (*_backward(*ctx.saved_tensors, plan, g_y, groups, act, need[0], need[1], need[2]), None, None, None)


def group_norm(x: Tensor, groups: int, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5,
               activation: str = "identity") -> Tensor:
    """Group norm of x [B, C, H, W] (float32, bfloat16 or float16) followed by ``activation``
    ("identity", "relu", "sigmoid" or "silu"): y of x's dtype, channels last.

    weight, bias: [C], float32 in the kernels (other floating types are widened, their gradients
    narrowed), or None. A channels-last x, and a slice of one along batch or channels, is read in
    place; any other layout is copied once. Gradients with respect to x, weight and bias; second derivatives and
    forward-mode derivatives are refused.
    """
    if activation not in ACTIVATIONS:
        raise _lib.ProtosegError(f"activation {activation!r} has no HIP kernel (one of {sorted(ACTIVATIONS)})")
    if not eps >= 0:
        raise _lib.ProtosegError(f"group norm eps {eps}")
    _lib.refuse_tangents("group norm", x, weight, bias)
    if weight is not None and weight.dtype != torch.float32 and weight.is_floating_point():
        weight = weight.float()
    if bias is not None and bias.dtype != torch.float32 and bias.is_floating_point():
        bias = bias.float()
    args = (x, weight, bias, int(groups), float(eps), ACTIVATIONS[activation])
    if not _lib.direct(x, weight, bias):
        _lib.require_device(x, weight, bias)
        return torch.ops.protoseg.group_norm(*args)[0]
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
