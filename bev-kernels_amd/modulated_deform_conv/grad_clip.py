"""The norm of all gradients together and their clipping to a largest norm: what comes between
the backward passes of the layers and the optimizer. A few launches for all tensors, of any
mixture of types, on the kernels of libbevk.so. The reference has no counterpart."""
from __future__ import annotations

import torch


def _ext():
    import _modulated_deform_conv_ext as ext
    return ext


def _listed(tensors):
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def grad_norm(grads):
    """The 2-norm of all values of the tensors together: a 0-dim float32 tensor on their device
    (zero on the CPU for no tensors). Squares are summed in 64 bits, in one order. The tensors are on
    a GPU, in fp32 / fp16 / bf16; no gradient flows through the norm."""
    grads = _listed(grads)
    return _ext().clip_gradients(grads) if grads else torch.zeros(())


def clip_gradients_(grads, max_norm, out=None):
    """Scales all gradients by min(1, max_norm / (norm + 1e-6)) and returns their norm before that
    (a 0-dim float32 tensor; nothing waits for it). In place, or into the tensors ``out`` of the
    same shapes and strides, for instance fp32 gradients for the optimizer from 16-bit ones.
    fp32 / fp16 / bf16, dense in memory. Each tensor once: overlapping outputs are refused.
    A norm of Inf or NaN goes through as in torch.nn.utils.clip_grad_norm_ (test the returned
    norm before the optimizer's step)."""
    grads = _listed(grads)
    out = None if out is None else _listed(out)
    if not max_norm >= 0:
        raise RuntimeError(f"clip_gradients_: max_norm must not be negative, got {max_norm}")
    if not grads:
        if out:
            raise RuntimeError(f"clip_gradients: {len(out)} outputs for 0 gradients")
        return torch.zeros(())
    return _ext().clip_gradients(grads, max_norm, out)


def clip_grad_norm_(parameters, max_norm):
    """clip_gradients_ on the .grad of the parameters that have one, in place, as
    torch.nn.utils.clip_grad_norm_ with its default norm."""
    return clip_gradients_([p.grad for p in _listed(parameters) if p.grad is not None], max_norm)
