"""Group normalization with an activation on channels-last maps, the norm of layers whose batch
is too small for batch statistics, beside the FrozenBN + ReLU epilogue of dcn_split_nhwc.

Forward and backward run on the kernels of libbevk.so: sums in 64 bits, everything else in
32, rounded once to the input's type. The reference has no counterpart."""
from __future__ import annotations

import torch
import torch.nn as nn

import _bevk as _b

_loaded = None


def _ext():
    global _loaded
    if _loaded is None:
        import _modulated_deform_conv_ext
        _loaded = _modulated_deform_conv_ext
    return _loaded


def _dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


class GroupNormActNHWCFunction(torch.autograd.Function):
    """y = act(group_norm(x)) for x [N, ..., C]; gradients flow to x, weight and bias."""

    @staticmethod
    def forward(ctx, x_nhwc, num_groups, weight, bias, eps, act):
        x, weight, bias = _dense(x_nhwc), _dense(weight), _dense(bias)
        y, stats, ctx.sizes = _ext()._group_norm_run(x, num_groups, weight, bias, eps, act)
        ctx.save_for_backward(x, weight, bias, stats)
        return y

    @staticmethod
    @_b.once_differentiable
    def backward(ctx, grad_y):
        x, weight, bias, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        grad_x, grad_w, grad_b = _ext()._group_norm_gradients(
            _dense(grad_y), x, weight, bias, stats, (need[0], need[2], need[3]), ctx.sizes)
        return grad_x, None, grad_w, grad_b, None, None


def group_norm_act_nhwc(x_nhwc, num_groups, weight=None, bias=None, eps=1e-5, act=None):
    """act(group norm of x_nhwc [N, ..., C]) over the positions and the C / num_groups channels of
    each group; weight and bias [C] in the input's type or float32 (or None: 1 and 0); act None,
    "relu" or "silu". fp32 / fp16 / bf16. Differentiable once, in reverse mode."""
    if _b.records_nothing():  # (without the bookkeeping of a Function, 4 us of a small call)
        return _ext()._group_norm_run(_dense(x_nhwc), num_groups, _dense(weight), _dense(bias), eps, act,
                                      False)[0]
    return GroupNormActNHWCFunction.apply(x_nhwc, num_groups, weight, bias, eps, act)


class GroupNormAct2d(nn.Module):
    """Group normalization and activation of x [N, C, H, W]; parameters named as nn.GroupNorm's.
    A channels_last input is a free NHWC view and the output keeps the input's memory format, as
    in dcn_apply_nchw."""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, act="relu"):
        super().__init__()
        if num_channels % num_groups != 0:
            raise ValueError("num_channels must be divisible by num_groups")
        if act not in (None, "relu", "silu"):
            raise ValueError("act must be None, 'relu' or 'silu'")
        self.num_groups, self.num_channels, self.eps, self.act = num_groups, num_channels, eps, act
        self.weight = nn.Parameter(torch.ones(num_channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(num_channels)) if affine else None

    def forward(self, x):
        if x.dim() != 4:
            raise ValueError(f"Expected 4D tensor as input, got {x.dim()}D tensor instead.")
        is_cl = x.is_contiguous(memory_format=torch.channels_last)
        y = group_norm_act_nhwc(x.permute(0, 2, 3, 1), self.num_groups, self.weight, self.bias,
                                self.eps, self.act).permute(0, 3, 1, 2)
        return y if is_cl else y.contiguous()

    def extra_repr(self):
        return (f"{self.num_groups}, {self.num_channels}, eps={self.eps}, "
                f"affine={self.weight is not None}, act={self.act!r}")
