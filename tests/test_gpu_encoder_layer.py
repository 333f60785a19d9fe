"""A layer of the bird's-eye-view encoder with the operators in a row: value and attention projections,
deformable attention, output projection, norm onto the residual, feed-forward layer with its activation and
residual, gated norm; backward, the gradients' norm and an AdamW step. Against the same layer of elementary
torch operations around the same attention in fp32.

Bounds in the 2-norm of a tensor: in fp32 each of the twelve operators in a row is within 2^-16 of its result
by its own tests' bounds at these sizes, 12 * 2^-16; in 16 bits each rounds its result to half a step e at
most and passes on what it was given at most doubled in all (norms and projections of unit scale), 24 e."""
import functools

import pytest
import torch
import torch.nn.functional as F

import modulated_deform_conv as mdc
import msda_opt2

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, W, C, HIDDEN = 20, 21, 256, 512
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _layer(dtype, seed):
    g = torch.Generator().manual_seed(seed)

    def rand(*s, scale=1.0, mean=0.0):
        return (mean + scale * torch.randn(*s, generator=g)).to(dtype).to(DEV)

    params = {"wv": rand(C, C, scale=C ** -0.5), "bv": rand(C, scale=0.1), "wa": rand(32, C, scale=0.5 * C ** -0.5),
              "wo": rand(C, C, scale=C ** -0.5), "bo": rand(C, scale=0.1), "n1w": rand(C, scale=0.1, mean=1.0),
              "n1b": rand(C, scale=0.1), "w1": rand(HIDDEN, C, scale=C ** -0.5), "b1": rand(HIDDEN, scale=0.1),
              "w2": rand(C, HIDDEN, scale=HIDDEN ** -0.5), "b2": rand(C, scale=0.1),
              "gate": rand(C, scale=0.2, mean=1.0), "n2w": rand(C, scale=0.1, mean=1.0), "n2b": rand(C, scale=0.1)}
    loc = torch.rand(1, H * W, 8, 1, 4, 2, generator=g).to(dtype).to(DEV)
    return params, rand(1, H * W, C), loc, rand(1, H * W, C)


@functools.lru_cache(maxsize=None)
def _levels():
    """Sizes and starts of the one level (copied to the device once: not within a capture)."""
    return torch.tensor([[H, W]], device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)


def _attend(value, weights, loc):
    attn = torch.softmax(weights.view(1, H * W, 8, 4), -1).view(1, H * W, 8, 1, 4)
    return msda_opt2.multi_scale_deformable_attn(value.view(1, H * W, 8, 32), *_levels(), loc, attn)


def _ours(p, x, loc):
    linear, norm = msda_opt2.linear_act, msda_opt2.residual_norm
    a = _attend(linear(x, p["wv"], p["bv"]), linear(x, p["wa"]), loc)
    y = norm(linear(a, p["wo"], p["bo"]), x, p["n1w"], p["n1b"], with_stream=False)
    f = linear(linear(y, p["w1"], p["b1"], "gelu"), p["w2"], p["b2"], None, y)
    z, stream = norm(f, y, p["n2w"], p["n2b"], gate=p["gate"], scale=0.5)
    return z + 0.1 * stream


def _plain(p, x, loc):
    a = _attend(F.linear(x, p["wv"], p["bv"]), F.linear(x, p["wa"]), loc)
    y = F.layer_norm(x + F.linear(a, p["wo"], p["bo"]), (C,), p["n1w"], p["n1b"])
    f = F.linear(F.gelu(F.linear(y, p["w1"], p["b1"])), p["w2"], p["b2"]) + y
    stream = y + 0.5 * p["gate"] * f
    return F.layer_norm(stream, (C,), p["n2w"], p["n2b"]) + 0.1 * stream


def _off(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_layer_and_step(dtype):
    half = torch.finfo(TYPES[dtype]).eps / 2
    bound = 12 * 2.0 ** -16 if dtype == "fp32" else 24 * half
    params, x, loc, go = _layer(TYPES[dtype], 1)
    leaves = {n: v.clone().requires_grad_() for n, v in params.items()}
    out = _ours(leaves, x, loc)
    grads = torch.autograd.grad(out, list(leaves.values()), go)
    wide = {n: v.float().requires_grad_() for n, v in params.items()}
    ref = _plain(wide, x.float(), loc.float())
    ref_grads = torch.autograd.grad(ref, list(wide.values()), go.float())
    assert _off(out, ref) <= bound
    for n, a, b in zip(leaves, grads, ref_grads):
        assert a.shape == b.shape and a.dtype == TYPES[dtype] and _off(a, b) <= bound, n

    # the step on fp32 parameters with copies in the layer's type, against torch's from the same gradients
    master = [v.detach().float().clone() for v in params.values()]
    copies = [v.detach().clone() for v in params.values()]
    theirs = [torch.nn.Parameter(v.clone()) for v in master]
    opt = torch.optim.AdamW(theirs, lr=1e-3, weight_decay=0.01)
    state = mdc.adamw_state(master)
    norm = mdc.grad_norm(grads)
    for v, g in zip(theirs, grads):
        v.grad = g.float() * min(1.0, 2.0 / (norm.item() + 1e-6))
    for _ in range(2):
        mdc.adamw_step_(master, list(grads), state, lr=1e-3, norm=norm, max_norm=2.0, copies=copies)
        opt.step()
    for a, c, b in zip(master, copies, theirs):
        # two steps of at most 1e-3, each evaluated to 2^-20, and the sums' roundings
        assert ((a - b).abs() <= 2e-3 * 2.0 ** -18 + 4 * 2.0 ** -24 * b.abs()).all()
        assert torch.equal(c, a.to(c.dtype))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_training(bits):
    """Forward, backward, norm, step and the weights for the next forward in one graph, against the same
    eager; the attention's backward may add up in another order in fp32."""
    params, x, loc, go = _layer(torch.bfloat16, 2)

    def start():
        weights = [v.clone().requires_grad_() for v in params.values()]
        master = [v.detach().float().clone() for v in params.values()]
        return weights, master, mdc.adamw_state(master, bits, 3)

    def step(weights, master, state):
        out = _ours(dict(zip(params, weights)), x, loc)
        grads = torch.autograd.grad(out, weights, go)
        mdc.adamw_step_(master, list(grads), state, lr=1e-3, max_norm=1.0, copies=[w.detach() for w in weights])
        return out.detach()

    a, b = start(), start()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*a)
    torch.cuda.current_stream().wait_stream(side)
    step(*b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(*a)
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        want = step(*b)
        assert a[2]["step"].item() == b[2]["step"].item() == k + 2
        assert _off(held, want) <= 2.0 ** -8
        for p, q in zip(a[1], b[1]):  # a gradient's last bit decides about a code of a moment
            assert ((p - q).abs() <= 3e-3).all() and _off(p, q) <= 2.0 ** -8
