"""Embedding rows by index with a scale: the object queries of a decoder, learned positions, or
the cells of a bird's-eye-view grid that each camera sees (the cross-attention runs on those
alone, padded to one length). The attention beside it samples rows between positions; this
looks whole ones up. The reference has no counterpart."""
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


def _lookup(weight, index, scale, padding_idx):
    """The rows, and the index as it was read."""
    if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
        raise RuntimeError("embedding_lookup: padding_idx must be a row of the table, got "
                           f"{padding_idx}")
    if not index.is_contiguous():
        index = index.contiguous()
    if not weight.is_contiguous():
        weight = weight.contiguous()
    return _ext().embedding_forward(weight, index, scale), index


class EmbeddingLookupFunction(torch.autograd.Function):
    """out [*index.shape, D] = scale * weight[index]; the gradient flows to weight [V, D]."""

    @staticmethod
    def forward(ctx, weight, index, scale=1.0, padding_idx=None):
        out, index = _lookup(weight, index, scale, padding_idx)
        ctx.save_for_backward(index)
        ctx.args = weight.shape[0], scale, -1 if padding_idx is None else padding_idx
        return out

    @staticmethod
    @_b.once_differentiable
    def backward(ctx, grad_output):
        index, = ctx.saved_tensors
        if not grad_output.is_contiguous():
            grad_output = grad_output.contiguous()
        return _ext()._embedding_gradient(grad_output, index, *ctx.args), None, None, None


def embedding_lookup(weight, index, scale=1.0, padding_idx=None):
    """scale * weight[index]: weight [V, D] fp32 / fp16 / bf16, index int64 or int32 of any shape
    -> [*index.shape, D]. An index outside [0, V) (-1 in a padded list) gives a row of zeros and
    gets no gradient. The row padding_idx is looked up as any other, and its gradient is zero, as
    in torch.nn.Embedding. The gradient is dense, adds up in fp32 in a fixed order and is the same
    on every run. Differentiable once, in reverse mode."""
    if _b.records_nothing():  # (without the bookkeeping of a Function, 4 us of a small call)
        return _lookup(weight, index, scale, padding_idx)[0]
    return EmbeddingLookupFunction.apply(weight, index, scale, padding_idx)
