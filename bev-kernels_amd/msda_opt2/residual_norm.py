"""The norms between two blocks of a transformer layer: the attention's or the feed-forward layer's output
through a norm of its own or none, times a gate and a scale onto the residual stream, and the norm
that the next block reads. One pass over the data; forward and backward run on the kernels of
libbevk.so. The reference has no counterpart."""
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


class ResidualNormFunction(torch.autograd.Function):
    """(y, stream) of residual_norm; gradients flow to all tensors."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, gate, block_weight, block_bias, options):
        scale, block_norm, kind, eps, with_stream = options
        y, h, stats, ctx.sizes = _ext().residual_norm_forward(
            x, residual, weight, bias, gate, scale, (block_weight, block_bias) if block_norm else None, kind, eps,
            with_stream, True)
        ctx.options = options
        ctx.save_for_backward(x, residual, stats, weight, bias, gate, block_weight, block_bias)
        ctx.set_materialize_grads(False)
        return (y, h) if with_stream else y

    @staticmethod
    @_b.once_differentiable
    def backward(ctx, grad_y, grad_stream=None):
        x, residual, stats, weight, bias, gate, bw, bb = ctx.saved_tensors
        scale, block_norm, *_ = ctx.options
        if grad_y is None:
            if grad_stream is None:
                return (None,) * 8
            grad_y = torch.zeros_like(x)
        grads = _ext().residual_norm_backward(_dense(grad_y), _dense(grad_stream), x, residual, stats, weight, bias,
                                              gate, scale, (bw, bb) if block_norm else None, ctx.sizes,
                                              ctx.needs_input_grad)
        return (*grads, None)


def residual_norm(x, residual=None, weight=None, bias=None, gate=None, scale=1.0, block_norm=None, kind="layer",
                  eps=1e-5, with_stream=True):
    """(y, stream), or y alone without with_stream:

      p = x, or with block_norm=(weight, bias) the norm of x
      stream = residual + scale * gate * p
      y = the norm of the stream

    over the last dimension of x [..., C]; the norm is "layer" (v - mean) / sqrt(var + eps) * weight +
    bias or "rms" v / sqrt(mean of squares + eps) * weight + bias. A weight or bias of None is 1 or 0,
    a residual of None 0. gate: [C], or one for each first index of x ([B, C], or with ones between).
    fp32 / fp16 / bf16; weights and biases in the input's type or fp32 (all of one), the gate too.
    Sums are fp32; y and the gradients are those of the stream before its rounding. x and residual are
    kept for the backward, the stream is not. Differentiable once, in reverse mode; all gradients are
    the same on every run."""
    block_weight, block_bias = (None, None) if block_norm is None else block_norm
    x, residual, weight, bias, gate = _dense(x), _dense(residual), _dense(weight), _dense(bias), _dense(gate)
    if block_norm is not None:
        block_weight, block_bias = _dense(block_weight), _dense(block_bias)
    if _b.records_nothing():  # (without the bookkeeping of a Function)
        y, h, _, _ = _ext().residual_norm_forward(
            x, residual, weight, bias, gate, scale, None if block_norm is None else (block_weight, block_bias), kind,
            eps, with_stream)
        return (y, h) if with_stream else y
    return ResidualNormFunction.apply(x, residual, weight, bias, gate, block_weight, block_bias,
                                      (scale, block_norm is not None, kind, eps, with_stream))
