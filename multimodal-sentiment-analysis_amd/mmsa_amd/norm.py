"""Group normalisation with an activation over channels-last maps.

Stands where the audio branch's ``BatchNorm -> ReLU`` pairs stand (`CNN implementation/multimodal_model.py:48-66`) when
the batch of one GPU is too small for statistics over the batch: every sample is normalised by itself, so nothing in the
forward or backward pass depends on the other rows.  The formulas are ``torch.nn.GroupNorm``'s followed by the activation;
both are one operator here, so the normalised map is neither written nor read again.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib, ops


def _channels_last(x: torch.Tensor) -> torch.Tensor:
    """x [B, C, *positions] with its values in the order [B, *positions, C], one after another: x itself where it lies so
    already, else a copy."""
    if x.dim() == 4:
        return x if x.is_contiguous(memory_format=torch.channels_last) else x.contiguous(
            memory_format=torch.channels_last)
    rows = x.movedim(1, -1)
    return x if rows.is_contiguous() else rows.contiguous().movedim(-1, 1)


class _GroupNormActFn(torch.autograd.Function):
    """One node from the map as the caller holds it to the result; x is in channels-last memory already."""

    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        B, C = x.shape[:2]
        y = torch.empty_like(x)
        stats = torch.empty((B, groups, 2), dtype=torch.float64, device=x.device)
        P = math.prod(x.shape[2:])
        if y.numel():
            ops._group_norm_launch_fwd(x, weight, bias, y, stats, B, P, C, groups, eps, act)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.args = (B, P, C, groups, act)
        return y

    @staticmethod
    def _backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        want = ctx.needs_input_grad
        if not x.numel():
            return tuple(torch.zeros_like(t) if w else None for t, w in zip((x, weight, bias), want)) + (None,) * 3
        dx = torch.empty_like(x) if want[0] else None
        dw = torch.empty_like(weight) if want[1] else None
        db = torch.empty_like(bias) if want[2] else None
        ops._group_norm_launch_bwd(_channels_last(dy), x, weight, bias, stats, dx, dw, db, *ctx.args)
        return dx, dw, db, None, None, None

    @staticmethod
    def backward(ctx, dy):
        # the guard against a gradient of the gradient costs host time, and only a graph of the backward pass needs it
        return (_guarded if torch.is_grad_enabled() else _GroupNormActFn._backward)(ctx, dy)


_guarded = once_differentiable(_GroupNormActFn._backward)


def group_norm_act(x: torch.Tensor, num_groups: int, weight=None, bias=None, eps: float = 1e-5,
                   activation: str = "none") -> torch.Tensor:
    """``activation(group_norm(x, num_groups, weight, bias, eps))`` for x [B, C, *positions] on the GPU.

    float32, bfloat16 or float16 maps; ``weight`` / ``bias`` [C] float32 or None; activation "none", "relu", "silu" or
    "gelu" (erf form).  Maps in channels-last memory (what the convolutions here return) are used as they lie, others
    are copied into that order; the result is in channels-last memory.  Statistics and parameter gradients are held in
    32 bits or more whatever the map's type.  Gradients flow to x, weight and bias (once: no gradient of a gradient; no
    forward-mode derivatives).
    """
    if x.dim() < 2:
        raise ValueError("group_norm_act: x must be [B, C, *positions]")
    if not x.is_cuda:
        raise _lib.MmsaError("group_norm_act: x must live on the GPU (the HIP kernels have no CPU path)")
    if x.dtype not in ops.DTYPE_CODES:
        raise TypeError(f"group_norm_act: float32, bfloat16 or float16 maps, got {x.dtype}")
    B, C = x.shape[:2]
    ops._group_norm_check(C, num_groups, activation, weight, bias, x.get_device())
    x = _channels_last(x)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _GroupNormActFn.apply(x, weight, bias, num_groups, eps, activation)
    # a dual tensor asks for no gradient; past the node, which refuses it, its tangent would get lost without a word (the
    # level is asked first, where torch has it: three tensors unpacked are a microsecond)
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (x, weight, bias)):
        raise NotImplementedError("group_norm_act has no forward-mode derivative (jvp)")
    y = torch.empty_like(x)
    if y.numel():
        ops._group_norm_launch_fwd(x, weight, bias, y, None, B, math.prod(x.shape[2:]), C, num_groups, eps, activation)
    return y


class GroupNormAct(nn.Module):
    """``torch.nn.GroupNorm`` followed by an activation as one operator: same constructor order, parameters and
    ``state_dict`` keys (``weight``, ``bias``) as ``nn.GroupNorm``; see :func:`group_norm_act`.  A module converted to
    16 bits keeps its parameters in that type and computes with their float32 values."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, affine: bool = True,
                 activation: str = "relu"):
        super().__init__()
        if num_groups < 1 or num_channels % num_groups:
            raise ValueError("num_channels must be divisible by num_groups")
        if activation not in ops.ACTIVATIONS:
            raise ValueError(f"activation {activation!r} is none of {', '.join(ops.ACTIVATIONS)}")
        self.num_groups, self.num_channels, self.eps, self.activation = num_groups, num_channels, eps, activation
        self.weight = nn.Parameter(torch.ones(num_channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(num_channels)) if affine else None

    def forward(self, x):
        if x.dim() < 2 or x.shape[1] != self.num_channels:
            raise ValueError(f"GroupNormAct({self.num_groups}, {self.num_channels}) got a map of shape {tuple(x.shape)}")
        # the kernels take float32 parameters; those of a module converted to 16 bits are widened (C values each)
        weight, bias = (p if p is None or p.dtype not in (torch.bfloat16, torch.float16) else p.float()
                        for p in (self.weight, self.bias))
        return group_norm_act(x, self.num_groups, weight, bias, self.eps, self.activation)

    def extra_repr(self):
        return (f"{self.num_groups}, {self.num_channels}, eps={self.eps}, affine={self.weight is not None}, "
                f"activation={self.activation!r}")
