"""The optimizer's step behind the clipping: AdamW over all tensors of a model in a few launches, on
the kernels of libbevk.so, with moments in 32 bits or in 8. The reference has no counterpart."""
from __future__ import annotations

import torch

from .grad_clip import _listed, grad_norm


def _ext():
    import _modulated_deform_conv_ext as ext
    return ext


def adamw_state(params, bits=32, seed=0):
    """A new state of adamw_step_ for these parameters: a dict of tensors on their device that may be
    saved and loaded as it is.

    exp_avg, exp_avg_sq   the moments of all parameters in a row, each parameter's part at a multiple
                          of 128 values: float32 zeros, or with bits=8 uint8 codes
    exp_avg_scale, exp_avg_sq_scale   (8 bits) a scale for each 128 values
    step                  int64, the steps so far
    seed                  of the random rounding of 8-bit moments; a number

    8 bits: 128 values share an exponent, each has 3 mantissa bits and a range of 2^16 (first
    moment, which loses what is below it) or 2^31 (second moment, which holds it at the least)
    below the largest, and is rounded at random. Same seed, steps and gradients: the same results."""
    params = _listed(params)
    if bits not in (8, 32):
        raise RuntimeError(f"adamw_state: moments have 8 or 32 bits, got {bits}")
    if not params:
        raise RuntimeError("adamw_state: no parameters")
    if not 0 <= seed < 2 ** 64:
        raise RuntimeError(f"adamw_state: seed must be in [0, 2^64), got {seed}")
    ext, device = _ext(), params[0].device
    total = ext.adamw_values(params)
    dtype = torch.float32 if bits == 32 else torch.uint8
    state = {"exp_avg": torch.zeros(total, dtype=dtype, device=device),
             "exp_avg_sq": torch.zeros(total, dtype=dtype, device=device)}
    if bits == 8:
        for name in ("exp_avg_scale", "exp_avg_sq_scale"):
            state[name] = torch.full((total // ext.ADAMW_BLOCK,), 32, dtype=torch.uint8, device=device)
    state["step"] = torch.zeros(1, dtype=torch.int64, device=device)
    state["seed"] = seed
    return state


def adamw_step_(params, grads, state, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, norm=None,
                max_norm=None, copies=None):
    """One AdamW step on all parameters, in place, as torch.optim.AdamW's:

      g = min(1, max_norm / (norm + 1e-6)) * grad        (with max_norm)
      m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
      p = (1 - lr weight_decay) p - lr / (1 - beta1^t) * m / (sqrt(v / (1 - beta2^t)) + eps)

    params, grads: lists of tensors of the same shapes and strides, fp32 / fp16 / bf16 in any mixture,
    dense in memory, on one GPU; arithmetic in fp32, each result rounded once (16-bit parameters lose
    updates below half their step: keep fp32 ones and have the model's 16-bit weights as copies).
    state: of adamw_state for the same parameters in the same order; one step at a time may use it.
    lr: a number, or one float32 on the device, for schedules under graph replay.
    max_norm: gradients are clipped by the norm of all of them on the way, without being written:
    norm, a float32 on the device from grad_norm, or None, and it is computed here.
    copies: tensors that receive the new parameters in their own type.
    eps may be 0: where v is 0 too (never used, or a gradient below 1e-21) a value only decays.
    Nothing waits for the device; a captured step counts on at every replay. A gradient of Inf or NaN
    goes through as in torch.optim.AdamW (with 8-bit moments into the 128 values around it): test
    the norm before the step. The same results on every run."""
    params, grads = _listed(params), _listed(grads)
    copies = None if copies is None else _listed(copies)
    if len(grads) != len(params):
        raise RuntimeError(f"adamw_step_: {len(grads)} gradients for {len(params)} parameters")
    if not params:
        raise RuntimeError("adamw_step_: no parameters")
    for k, g in enumerate(grads):
        if g is None:
            raise RuntimeError(f"adamw_step_: parameter {k} has no gradient; give zeros, or leave it out of the state")
    if norm is not None and max_norm is None:
        raise RuntimeError("adamw_step_: norm without max_norm")
    if max_norm is not None and norm is None:
        norm = grad_norm(grads)
    _ext().adamw_step(params, grads, state, lr, *betas, eps, weight_decay, norm,
                      0.0 if max_norm is None else max_norm, copies)


def adamw_moments(state, dtype=torch.float32):
    """(exp_avg, exp_avg_sq) of a state as values in a row (parameter k's begin at the sum of the
    sizes before it, each rounded up to 128): the state's own tensors where they have that type. 8-bit
    moments are given in float32 or bfloat16, exactly."""
    return _ext().adamw_moments(state, dtype)
