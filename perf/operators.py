"""The work that programs have the training-side operators do, as cases to measure.

Three operators that stand beside the deformable layers and the attention of this library:

* group normalization with an activation on channels-last maps (``group_norm_act_nhwc``),
  which follows a convolution of a detection head or brings feature levels to one width
  before multi-scale attention: forward, and the training step;
* the lookup of embedding rows with a scale (``embedding_lookup``): object queries, cells
  of a bird's-eye-view grid picked for each camera (padded with -1), tokens of a
  vocabulary; forward, and the training step, whose gradient adds up the rows of equal
  indices;
* the global norm of a model's gradients and their clipping (``clip_gradients_``), the step
  between the backward pass and the optimizer, into the buffer of fp32 gradients that the
  optimizer reads.

With ``own`` false a pass computes the plain form in elementary torch operations, with it
true the library's call. ``listed()`` gives the cases, ``draw`` one more of the same ranges,
``prepare`` / ``run`` one pass as a program calls it, ``exact`` the same outputs in 64 bits.
"""
from __future__ import annotations

import math
import os
import sys

import torch
import torch.nn.functional as F

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "bev-kernels_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


# ---------------------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------------------

def _norm(name, batch, h, w, channels, groups, act, dtype, train=False):
    return {"name": name, "op": "norm", "batch": batch, "h": h, "w": w, "channels": channels,
            "groups": groups, "act": act, "dtype": dtype, "train": train}


def _lookup(name, kind, rows, dim, sets, length, dtype, train=False):
    return {"name": name, "op": "lookup", "kind": kind, "rows": rows, "dim": dim, "sets": sets,
            "length": length, "dtype": dtype, "train": train}


def _clip(name, rows, width, layers, max_norm, dtype):
    return {"name": name, "op": "clip", "rows": rows, "width": width, "layers": layers,
            "max_norm": max_norm, "dtype": dtype}


def listed():
    return [
        # The coarsest feature level of one camera at inference. The smallest call.
        _norm("norm_15x25_fp32", 1, 15, 25, 256, 32, "relu", "fp32"),
        # A head's convolution over the res4 maps of six cameras at inference.
        _norm("norm_res4_fp16", 6, 58, 100, 256, 32, "relu", "fp16"),
        # The finest level of six cameras, the largest map there is.
        _norm("norm_fine_bf16", 6, 116, 200, 256, 32, "silu", "bf16"),
        # Training step of a head on res4 in bf16.
        _norm("norm_res4_train_bf16", 6, 58, 100, 256, 32, "relu", "bf16", train=True),
        # Training step on the res5 maps in fp32, groups of 16 channels, no activation (the
        # projection of a level before the attention).
        _norm("norm_res5_train_fp32", 6, 29, 50, 512, 32, "none", "fp32", train=True),
        # A decoder's 300 object queries for one image.
        _lookup("lookup_queries_fp32", "queries", 300, 256, 1, 300, "fp32"),
        # Cells of a 200 x 200 grid that six cameras see, padded to 10,000 a camera: the
        # queries of the camera cross-attention in a training step.
        _lookup("lookup_cameras_train_fp16", "cameras", 40000, 256, 6, 10000, "fp16",
                train=True),
        # A language model's tokens at inference and in a training step.
        _lookup("lookup_tokens_bf16", "tokens", 32768, 2048, 4, 4096, "bf16"),
        _lookup("lookup_tokens_train_bf16", "tokens", 32768, 1024, 8, 2048, "bf16", train=True),
        # The gradients of one small layer: few tensors, where launches count.
        _clip("clip_layer_fp32", 0, 128, 1, 35.0, "fp32"),
        # An encoder of six layers with its grid of queries, mixed with 16-bit gradients.
        _clip("clip_encoder_bf16", 40000, 256, 6, 35.0, "bf16"),
        # A large model's gradients in fp32, norm above the limit.
        _clip("clip_model_fp32", 32768, 1024, 6, 1.0, "fp32"),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case: any operator, direction and type above at other sizes."""
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    op = rng.choice(["norm", "norm", "lookup", "lookup", "clip"])
    if op == "norm":
        train = rng.random() < 0.5
        channels, groups = rng.choice([(256, 32), (512, 32), (64, 8), (128, 32), (96, 32),
                                       (256, 256), (320, 32), (100, 25), (75, 5), (256, 1)])
        h, w = _log(rng, 7, 116), _log(rng, 7, 200)
        batch = rng.randint(1, 6)
        act = rng.choice(["none", "relu", "silu"])
        limit = 6 * 116 * 200 * 256 // (4 if train else 1) // (2 if dtype == "fp32" else 1)
        while batch * h * w * channels > limit:
            h, w = h - h // 8, w - w // 8
        return _unnamed(_norm("", batch, h, w, channels, groups, act, dtype, train))
    if op == "lookup":
        train = rng.random() < 0.5
        kind = rng.choice(["queries", "cameras", "tokens"])
        if kind == "queries":
            rows, dim, sets = _log(rng, 100, 2000), rng.choice([128, 256, 512]), rng.randint(1, 4)
            return _unnamed(_lookup("", kind, rows, dim, sets, rows, dtype, train))
        if kind == "cameras":
            side = rng.randint(50, 200)
            dim, sets = rng.choice([128, 256, 256]), rng.randint(1, 6)
            length = _log(rng, 200, side * side // 4)
            return _unnamed(_lookup("", kind, side * side, dim, sets, length, dtype, train))
        rows, dim = _log(rng, 1000, 65536), rng.choice([256, 320, 500, 512, 1001, 1024, 2048])
        sets, length = rng.randint(1, 8), _log(rng, 1, 4096)
        while (rows + 2 * sets * length) * dim * (2 if dtype == "fp32" else 1) > 3 * 2 ** 25:
            rows, length = rows - rows // 4, length - length // 4
        return _unnamed(_lookup("", kind, rows, dim, sets, length, dtype, train))
    width = rng.choice([64, 100, 128, 256, 320, 512, 1000, 1024])
    layers = _log(rng, 1, 12) if width < 1000 else _log(rng, 1, 5)
    rows = rng.choice([0, 300, _log(rng, 1000, 32768)])
    return _unnamed(_clip("", rows, width, layers, rng.choice([0.1, 1.0, 35.0]), dtype))


def _unnamed(case):
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------

def _norm_inputs(case, rand):
    """x as a convolution leaves it: each channel with a mean and a spread of its own."""
    n, h, w, c = (case[k] for k in ("batch", "h", "w", "channels"))
    dt = DTYPES[case["dtype"]]
    x = rand(n, h, w, c) * (0.5 + rand(c).abs()) + 0.5 * rand(c)
    s = {"x": x.to(dt), "weight": (1 + 0.2 * rand(c)).to(dt), "bias": (0.2 * rand(c)).to(dt)}
    if case["train"]:
        s["grad"] = rand(n, h, w, c).to(dt)
    return s


def _lookup_index(case, uniform):
    rows, sets, length = case["rows"], case["sets"], case["length"]
    if case["kind"] == "queries":  # every query once, for each image
        return torch.arange(length, device=DEV).repeat(sets, 1)
    if case["kind"] == "tokens":  # frequency falls as one over the rank
        u = uniform(sets, length).double()
        return (torch.exp(u * math.log(rows + 1)).long() - 1).clamp(0, rows - 1)
    # each camera sees a part of the cells; shorter lists are padded with -1
    index = uniform(sets, rows).argsort(1)[:, :length].sort(1).values
    seen = (length * (0.6 + 0.4 * uniform(sets, 1))).long()
    return torch.where(torch.arange(length, device=DEV) < seen, index, -1)


def _scale(case):
    return case["dim"] ** 0.5 if case["kind"] == "tokens" else 1.0


def _clip_shapes(case):
    """An embedding table or none, then for each layer four square matrices with their
    biases, two matrices of four times the width, and two norms."""
    d = case["width"]
    layer = [(d, d), (d,)] * 4 + [(4 * d, d), (4 * d,), (d, 4 * d), (d,)] + [(d,)] * 4
    shapes = ([(case["rows"], d)] if case["rows"] else []) + layer * case["layers"]
    return shapes


def _clip_inputs(case, rand):
    """Gradients of a spread of 0.01, one tensor each, and the fp32 buffer with room for all,
    each tensor's part at a multiple of 64 values."""
    grads = [(0.01 * rand(*s)).to(DTYPES[case["dtype"]]) for s in _clip_shapes(case)]
    sizes = [-(-g.numel() // 64) * 64 for g in grads]
    flat = torch.zeros(sum(sizes), device=DEV)
    out = [p[:g.numel()].view(g.shape) for p, g in zip(flat.split(sizes), grads)]
    return {"grads": grads, "flat": flat, "out": out}


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def rand(*size):
        return torch.randn(*size, device=DEV, generator=gen)

    def uniform(*size):
        return torch.rand(*size, device=DEV, generator=gen)

    if case["op"] == "norm":
        s = _norm_inputs(case, rand)
        if case["train"]:
            for k in ("x", "weight", "bias"):
                s[k].requires_grad_()
    elif case["op"] == "lookup":
        dt = DTYPES[case["dtype"]]
        s = {"weight": (rand(case["rows"], case["dim"]) / case["dim"] ** 0.5).to(dt),
             "index": _lookup_index(case, uniform)}
        if case["train"]:
            s["weight"].requires_grad_()
            s["grad"] = rand(*s["index"].shape, case["dim"]).to(dt)
    else:
        s = _clip_inputs(case, rand)
    return dict(s, case=case)


# ---------------------------------------------------------------------------------------
# One pass: the library's calls, or the plain form
# ---------------------------------------------------------------------------------------

def run(state):
    """The outputs; for a training step also the gradients."""
    case = state["case"]
    form = {"norm": (_norm_plain, _norm_own), "lookup": (_lookup_plain, _lookup_own),
            "clip": (_clip_plain, _clip_own)}[case["op"]]
    return form[1](state, case) if own else form[0](state, case)


def _norm_own(s, case):
    from modulated_deform_conv import group_norm_act_nhwc
    act = None if case["act"] == "none" else case["act"]
    args = (s["x"], case["groups"], s["weight"], s["bias"], EPS, act)
    if not case["train"]:
        with torch.no_grad():
            return [group_norm_act_nhwc(*args)]
    y = group_norm_act_nhwc(*args)
    return [y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["grad"])]


def _lookup_own(s, case):
    from msda_opt2 import embedding_lookup
    if not case["train"]:
        with torch.no_grad():
            return [embedding_lookup(s["weight"], s["index"], _scale(case))]
    out = embedding_lookup(s["weight"], s["index"], _scale(case))
    return [out.detach(), *torch.autograd.grad(out, s["weight"], s["grad"])]


def _clip_own(s, case):
    from modulated_deform_conv import clip_gradients_
    return [clip_gradients_(s["grads"], case["max_norm"], out=s["out"]), s["flat"]]


@torch.no_grad()
def _norm_plain(s, case):
    x = s["x"].float()
    n, h, w, c = x.shape
    per = c // case["groups"]
    weight, bias = s["weight"].float().view(-1, per), s["bias"].float().view(-1, per)
    x = x.view(n, h * w, -1, per)
    mean = x.mean((1, 3), keepdim=True)
    d = x - mean
    rstd = torch.rsqrt(d.square().mean((1, 3), keepdim=True) + EPS)
    xh = d * rstd
    z = xh * weight + bias
    if case["act"] == "relu":
        y = z.clamp(min=0)
    elif case["act"] == "silu":
        sig = 1 / (1 + torch.exp(-z))
        y = z * sig
    else:
        y = z
    y = y.view(n, h, w, c).to(s["x"].dtype)
    if not case["train"]:
        return [y]
    g = s["grad"].float().view(x.shape)
    if case["act"] == "relu":  # next to zero the sign of z takes 64 bits
        x64 = x.double()
        d64 = x64 - x64.mean((1, 3), keepdim=True)
        z64 = d64 / torch.sqrt(d64.square().mean((1, 3), keepdim=True) + EPS) * weight + bias
        g = g * (z64 > 0)
    elif case["act"] == "silu":
        g = g * (sig * (1 + z * (1 - sig)))
    gw = g * weight
    m1, m2 = gw.mean((1, 3), keepdim=True), (gw * xh).mean((1, 3), keepdim=True)
    gx = rstd * (gw - m1 - xh * m2)
    dt = s["x"].dtype
    return [y, gx.view(n, h, w, c).to(dt), (g * xh).sum((0, 1)).view(c).to(dt),
            g.sum((0, 1)).view(c).to(dt)]


@torch.no_grad()
def _lookup_plain(s, case):
    weight, index = s["weight"], s["index"]
    there = (index >= 0).unsqueeze(-1)
    rows = index.clamp(min=0)
    out = (weight[rows].float() * _scale(case) * there).to(weight.dtype)
    if not case["train"]:
        return [out]
    grad = torch.zeros(weight.shape, device=DEV)
    grad.index_add_(0, rows.flatten(), (s["grad"].float() * there).flatten(0, -2))
    return [out, (grad * _scale(case)).to(weight.dtype)]


@torch.no_grad()
def _clip_plain(s, case):
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    by = (case["max_norm"] / (norm + 1e-6)).clamp(max=1)
    [o.copy_(g.float() * by) for o, g in zip(s["out"], s["grads"])]
    return [norm, s["flat"]]


# ---------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------

def _rows_seen(case):
    """How many different rows a lookup reads, on average."""
    rows, n = case["rows"], case["sets"] * case["length"]
    if case["kind"] == "queries":
        return rows
    if case["kind"] == "cameras":
        return rows * (1 - (1 - 0.8 * case["length"] / rows) ** case["sets"])
    rank = torch.arange(1, rows + 1, dtype=torch.float64)
    p = torch.log((rank + 1) / rank) / math.log(rows + 1)
    return float((1 - (1 - p) ** n).sum())


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        n = case["batch"] * case["h"] * case["w"] * case["channels"]
        if not case["train"]:
            return {"bytes": size * (2 * n + 2 * case["channels"]), "flops": 9.0 * n}
        # forward, then x and the output's gradient read and a gradient written
        return {"bytes": size * (5 * n + 5 * case["channels"]), "flops": 24.0 * n}
    if case["op"] == "lookup":
        n, dim = case["sets"] * case["length"], case["dim"]
        ahead = 8 * n + size * dim * (_rows_seen(case) + n)
        if not case["train"]:
            return {"bytes": ahead, "flops": float(n * dim)}
        return {"bytes": ahead + 8 * n + size * dim * (n + case["rows"]),
                "flops": 3.0 * n * dim}
    n = sum(math.prod(s) for s in _clip_shapes(case))
    return {"bytes": (size + 4) * n + 4, "flops": 3.0 * n}


# ---------------------------------------------------------------------------------------
# The same in 64 bits
# ---------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        leaves = [s[k].detach().double().requires_grad_() for k in ("x", "weight", "bias")]
        planes = leaves[0].permute(0, 3, 1, 2).contiguous()
        y = F.group_norm(planes, case["groups"], leaves[1], leaves[2], EPS)
        y = {"relu": F.relu, "silu": F.silu, "none": lambda t: t}[case["act"]](y)
        y = y.permute(0, 2, 3, 1).contiguous()
        if not case["train"]:
            return [y.detach()]
        return [y.detach(), *torch.autograd.grad(y, leaves, s["grad"].double())]
    if case["op"] == "lookup":
        table = s["weight"].detach().double()
        known = torch.cat([table * _scale(case), table.new_zeros(1, case["dim"])])
        pick = torch.where(s["index"] < 0, case["rows"], s["index"])
        if not case["train"]:
            return [known[pick]]
        known.requires_grad_()
        out = F.embedding(pick, known)
        grad, = torch.autograd.grad(out, known, s["grad"].double())
        return [out.detach(), grad[:-1] * _scale(case)]
    squares = [torch.linalg.vector_norm(g.double()) ** 2 for g in s["grads"]]
    norm = torch.sqrt(sum(squares))
    by = min(1.0, case["max_norm"] / (norm.item() + 1e-6))
    flat = s["flat"].double()
    at = 0
    for g in s["grads"]:
        flat[at:at + g.numel()] = g.double().flatten() * by
        at += -(-g.numel() // 64) * 64
    return [norm, flat]
