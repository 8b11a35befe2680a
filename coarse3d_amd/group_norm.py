"""GroupNorm with a fused activation as an autograd function and a module, over ``ops.group_norm`` / ``ops.group_norm_bwd``.

What takes BatchNorm's place (salsanext_proto.py:46,50; projector.py:20) when a GPU trains on one or two range images: statistics
of one sample and one group of channels, the same in training and evaluation, with nothing to exchange between ranks."""
import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import ops


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act, slope):
        y, mean, rstd = ops.group_norm(x, groups, weight, bias, eps=eps, act=act, slope=slope)
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        ctx.act, ctx.slope = act, slope
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        dx, dw, db = ops.group_norm_bwd(dy.contiguous(), x, mean, rstd, weight, bias, act=ctx.act, slope=ctx.slope)
        return dx, dw, db, None, None, None, None


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, act="lrelu", slope=0.01):
    """act(GroupNorm(x)) over a channels-last tensor [N, ..., C] (``ops.group_norm``'s rules), differentiable once with respect to x,
    weight and bias."""
    return _GroupNormAct.apply(x, weight, bias, groups, eps, act, slope)


class GroupNormAct(nn.Module):
    """``nn.GroupNorm(num_groups, num_channels)`` followed by an activation, on [B, C, H, W] like the other modules here (stored
    channels last, as their outputs are, it is read in place).  act: "none", "lrelu" (``negative_slope``) or "silu".  State-dict keys
    as nn.GroupNorm: ``weight``, ``bias``."""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, act="lrelu", negative_slope=0.01):
        super().__init__()
        if num_groups < 1 or num_channels < 1 or num_channels % num_groups:
            raise ValueError(f"GroupNormAct: {num_channels} channels do not divide into {num_groups} groups")
        self.num_groups, self.num_channels, self.eps, self.act, self.negative_slope = num_groups, num_channels, eps, act, negative_slope
        self.weight = nn.Parameter(torch.ones(num_channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(num_channels)) if affine else None

    def extra_repr(self):
        return f"{self.num_groups}, {self.num_channels}, eps={self.eps}, affine={self.weight is not None}, act={self.act!r}"

    def forward(self, x):
        if x.dim() != 4 or x.shape[1] != self.num_channels:
            raise ValueError(f"GroupNormAct: expected [B, {self.num_channels}, H, W], got {tuple(x.shape)}")
        w, b = (None, None) if self.weight is None else (self.weight.float(), self.bias.float())      # (a module moved to 16 bits)
        y = group_norm_act(ops.to_nhwc(x), self.num_groups, w, b, self.eps, self.act, self.negative_slope)
        return ops.from_nhwc(y)
