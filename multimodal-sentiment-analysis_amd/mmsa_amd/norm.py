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
from torch.autograd.function import once_differentiable

from . import _lib, ops


def _rows(x: torch.Tensor) -> torch.Tensor:
    """[B, C, *positions] -> contiguous [B, P, C]; no copy for a map in channels-last memory."""
    B, C = x.shape[:2]
    if x.dim() == 4:
        return x.permute(0, 2, 3, 1).contiguous().view(B, x.shape[2] * x.shape[3], C)
    return x.movedim(1, -1).contiguous().view(B, math.prod(x.shape[2:]), C)


def _maps(rows: torch.Tensor, shape) -> torch.Tensor:
    """[B, P, C] -> [B, C, *positions] in channels-last memory."""
    if len(shape) == 4:
        return rows.view(shape[0], shape[2], shape[3], shape[1]).permute(0, 3, 1, 2)
    return rows.view(shape[0], *shape[2:], shape[1]).movedim(-1, 1)


class _GroupNormActFn(torch.autograd.Function):
    """One node from the map as the caller holds it to the result: the changes of layout are views made inside it."""

    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        rows = _rows(x)
        y = torch.empty_like(rows)
        stats = torch.empty((rows.shape[0], groups, 2), dtype=torch.float64, device=x.device)
        ops.group_norm_act_fwd(rows, weight, bias, y, stats, groups, eps, act)
        ctx.save_for_backward(rows, weight, bias, stats)
        ctx.groups, ctx.act, ctx.shape = groups, act, x.shape
        return _maps(y, x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        rows, weight, bias, stats = ctx.saved_tensors
        want = ctx.needs_input_grad
        dx = torch.empty_like(rows) if want[0] else None
        dw = torch.empty_like(weight) if want[1] else None
        db = torch.empty_like(bias) if want[2] else None
        ops.group_norm_act_bwd(_rows(dy), rows, weight, bias, stats, dx, dw, db, ctx.groups, ctx.act)
        return None if dx is None else _maps(dx, ctx.shape), dw, db, None, None, None


def group_norm_act(x: torch.Tensor, num_groups: int, weight=None, bias=None, eps: float = 1e-5,
                   activation: str = "none") -> torch.Tensor:
    """``activation(group_norm(x, num_groups, weight, bias, eps))`` for x [B, C, *positions] on the GPU.

    float32, bfloat16 or float16 maps; ``weight`` / ``bias`` [C] float32 or None; activation "none", "relu", "silu" or
    "gelu" (erf form).  Maps in channels-last memory (what the convolutions here return) are used as they lie, others
    are copied into that order; the result is in channels-last memory.  Statistics and parameter gradients are held in
    32 bits or more whatever the map's type.  Gradients flow to x, weight and bias (once: no gradient of a gradient).
    """
    if x.dim() < 2:
        raise ValueError("group_norm_act: x must be [B, C, *positions]")
    if not x.is_cuda:
        raise _lib.MmsaError("group_norm_act: x must live on the GPU (the HIP kernels have no CPU path)")
    B, C = x.shape[:2]
    if num_groups < 1 or C % num_groups or C < 1:
        raise ValueError(f"group_norm_act: {C} channels do not divide into {num_groups} groups")
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _GroupNormActFn.apply(x, weight, bias, num_groups, eps, activation)
    rows = _rows(x)
    y = torch.empty_like(rows)
    stats = torch.empty((B, num_groups, 2), dtype=torch.float64, device=x.device)
    ops.group_norm_act_fwd(rows, weight, bias, y, stats, num_groups, eps, activation)
    return _maps(y, x.shape)


class GroupNormAct(nn.Module):
    """``torch.nn.GroupNorm`` followed by an activation as one operator: same constructor order, parameters and
    ``state_dict`` keys (``weight``, ``bias``) as ``nn.GroupNorm``; see :func:`group_norm_act`."""

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
        return group_norm_act(x, self.num_groups, self.weight, self.bias, self.eps, self.activation)

    def extra_repr(self):
        return (f"{self.num_groups}, {self.num_channels}, eps={self.eps}, affine={self.weight is not None}, "
                f"activation={self.activation!r}")
