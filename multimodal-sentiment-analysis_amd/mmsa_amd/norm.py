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


class _GroupNormActFn(torch.autograd.Function):
    """x [B, P, C] contiguous -> y [B, P, C]."""

    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        y = torch.empty_like(x)
        stats = torch.empty((x.shape[0], groups, 2), dtype=torch.float64, device=x.device)
        ops.group_norm_act_fwd(x, weight, bias, y, stats, groups, eps, act)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.groups, ctx.act = groups, act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        want = ctx.needs_input_grad
        with torch.cuda.device(x.device):
            dx = torch.empty_like(x) if want[0] else None
            dw = torch.empty_like(weight) if weight is not None and want[1] else None
            db = torch.empty_like(bias) if bias is not None and want[2] else None
            ops.group_norm_act_bwd(dy.contiguous(), x, weight, bias, stats, dx, dw, db, ctx.groups, ctx.act)
        return dx, dw, db, None, None, None


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
    rows = x.movedim(1, -1)
    flat = rows.reshape(B, math.prod(x.shape[2:]), C).contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        y = _GroupNormActFn.apply(flat, weight, bias, num_groups, eps, activation)
    else:
        y = torch.empty_like(flat)
        stats = torch.empty((B, num_groups, 2), dtype=torch.float64, device=x.device)
        ops.group_norm_act_fwd(flat, weight, bias, y, stats, num_groups, eps, activation)
    return y.view(rows.shape).movedim(-1, 1)


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
