"""Projections with everything behind them: the value, output and feed-forward products around multi-scale
attention, with bias, activation and residual on the sums before their one rounding. Forward and
backward run on the kernels of libbevk.so. The reference has no counterpart."""
from __future__ import annotations

import torch

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


class LinearActFunction(torch.autograd.Function):
    """y = act(x W^T + b) + residual; gradients flow to all tensors."""

    @staticmethod
    def forward(ctx, x, weight, bias, act, residual):
        wanted = any(ctx.needs_input_grad[:3])  # (the residual's gradient is grad_y: nothing is kept for it)
        y, slope, ctx.sizes = _ext().linear_forward(x, weight, bias, act, residual, wanted)
        if wanted:
            ctx.save_for_backward(x, weight, bias, slope)
        return y

    @staticmethod
    @_b.once_differentiable
    def backward(ctx, grad_y):
        need = ctx.needs_input_grad
        grads = (None, None, None)
        if any(need[:3]):
            x, weight, bias, slope = ctx.saved_tensors
            grads = _ext().linear_backward(_dense(grad_y), x, weight, bias, slope, ctx.sizes, need[:3])
        return (*grads, None, grad_y if need[4] else None)


def linear_act(x, weight, bias=None, act=None, residual=None):
    """act(x @ weight.T + bias) + residual: x [..., K], weight [N, K], bias [N] in the input's type or
    float32 (or None), residual [..., N] (or None) -> [..., N]. fp32 / fp16 / bf16. act None, "relu",
    "silu" or "gelu" (z times the normal distribution below z, as torch's default). Everything behind the
    product is in fp32 and rounded once. SiLU and GELU, and ReLU with a residual, keep their
    derivative for the backward, as wide as the input (SiLU's and GELU's in 16 bits as int16). Differentiable once, in reverse mode; the same results on every run."""
    x, weight, bias, residual = _dense(x), _dense(weight), _dense(bias), _dense(residual)
    if _b.records_nothing():  # (without the bookkeeping of a Function)
        return _ext().linear_forward(x, weight, bias, act, residual)[0]
    return LinearActFunction.apply(x, weight, bias, act, residual)
