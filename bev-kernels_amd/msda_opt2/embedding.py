"""Embedding rows by index with a scale: the object queries of a decoder, learned positions, or
the cells of a bird's-eye-view grid that each camera sees (the cross-attention runs on those
alone, padded to one length). The attention beside it samples rows between positions; this
looks whole ones up. The reference has no counterpart."""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable


def _ext():
    import _modulated_deform_conv_ext
    return _modulated_deform_conv_ext


class EmbeddingLookupFunction(torch.autograd.Function):
    """out [*index.shape, D] = scale * weight[index]; the gradient flows to weight [V, D]."""

    @staticmethod
    def forward(ctx, weight, index, scale=1.0, padding_idx=None):
        if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
            raise RuntimeError("embedding_lookup: padding_idx must be a row of the table, got "
                               f"{padding_idx}")
        index = index.contiguous()
        out = _ext().embedding_forward(weight.contiguous(), index, scale)
        ctx.save_for_backward(index)
        ctx.num_embeddings, ctx.scale, ctx.padding_idx = weight.shape[0], scale, padding_idx
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        index, = ctx.saved_tensors
        grad = _ext().embedding_backward(grad_output.contiguous(), index, ctx.num_embeddings,
                                         ctx.scale, ctx.padding_idx)
        return grad, None, None, None


def embedding_lookup(weight, index, scale=1.0, padding_idx=None):
    """scale * weight[index]: weight [V, D] fp32 / fp16 / bf16, index int64 or int32 of any shape
    -> [*index.shape, D]. An index outside [0, V) (-1 in a padded list) gives a row of zeros and
    gets no gradient. The row padding_idx is looked up as any other, and its gradient is zero, as
    in torch.nn.Embedding. The gradient is dense, adds up in fp32 in a fixed order and is the same
    on every run. Differentiable once."""
    return EmbeddingLookupFunction.apply(weight, index, scale, padding_idx)
