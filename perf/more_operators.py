"""The operators of a transformer layer and its training step, as cases to measure.

Three operators that stand beside the attention, the norms and the clipping of this library:

* a projection with everything behind it (``linear_act``): y = act(x W^T + b) + residual, the
  values, outputs and feed-forward products around multi-scale attention; forward, and the
  training step with all gradients;
* the norms between two blocks (``residual_norm``): the block's output through a norm of its own
  (or none), times a gate and a scale onto the residual stream, and the next block's norm of that;
  forward, and the training step;
* an AdamW step over all tensors of a model (``adamw_step_``), with moments in 32 bits or in 8,
  gradients clipped by a norm that is there already, and 16-bit copies of the weights.

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
BLOCK = 128  # values of a moment that share a scale; each tensor's part begins at a multiple
LR, BETAS, ADAM_EPS, DECAY = 1e-4, (0.9, 0.999), 1e-8, 0.01


# ---------------------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------------------

def _linear(name, rows, k, n, act, residual, dtype, train=False):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "act": act,
            "residual": residual, "dtype": dtype, "train": train}


def _norm(name, sets, rows, channels, kind, gate, block_norm, stream, dtype, train=False):
    return {"name": name, "op": "norm", "sets": sets, "rows": rows, "channels": channels,
            "kind": kind, "gate": gate, "block_norm": block_norm, "stream": stream,
            "dtype": dtype, "train": train}


def _adamw(name, rows, width, layers, bits, grads, copies, max_norm):
    return {"name": name, "op": "adamw", "rows": rows, "width": width, "layers": layers,
            "bits": bits, "grads": grads, "copies": copies, "max_norm": max_norm}


def listed():
    return [
        # A decoder's 300 queries through the attention's output projection, onto the residual.
        _linear("linear_queries_fp16", 300, 256, 256, "none", True, "fp16"),
        # Four sequences that decode one token each, into a wide feed-forward layer.
        _linear("linear_decode_bf16", 4, 2048, 8192, "silu", False, "bf16"),
        # The value projection of all levels of six cameras.
        _linear("linear_values_fp16", 6 * 30825, 256, 256, "none", False, "fp16"),
        # The feed-forward layer of a 200 x 200 grid of queries in a training step.
        _linear("linear_ffn_train_bf16", 40000, 256, 512, "gelu", False, "bf16", train=True),
        # The output projection of that grid, in a training step in fp32.
        _linear("linear_output_train_fp32", 40000, 256, 256, "none", True, "fp32", train=True),
        # A wide feed-forward layer over 8 Ki tokens of a prompt.
        _linear("linear_prompt_bf16", 8192, 2048, 8192, "silu", False, "bf16"),
        # A decoder's 300 queries behind their attention. The smallest call.
        _norm("norm_queries_fp32", 1, 300, 256, "layer", "none", False, False, "fp32"),
        # The grid of queries behind the attention, at inference.
        _norm("norm_grid_bf16", 1, 40000, 256, "layer", "none", False, False, "bf16"),
        # Maps of six cameras whose blocks are gated by image, in a training step.
        _norm("norm_gated_train_fp16", 6, 5800, 512, "layer", "sets", False, True, "fp16",
              train=True),
        # 16 Ki tokens with a norm before and behind each block and a learned gate for each
        # channel, in a training step.
        _norm("norm_tokens_train_bf16", 8, 2048, 2048, "rms", "channels", True, True, "bf16",
              train=True),
        # An encoder of six layers with its grid of queries: 97 tensors, 15 M values.
        _adamw("adamw_encoder_32bit", 40000, 256, 6, 32, "fp32", False, 35.0),
        # A larger model in mixed precision: 8-bit moments, 16-bit gradients and weights.
        _adamw("adamw_model_8bit", 32768, 1024, 6, 8, "bf16", True, 0.0),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case: any operator, direction and type above at other sizes."""
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    op = rng.choice(["linear", "linear", "linear", "norm", "norm", "adamw"])
    if op == "linear":
        train = rng.random() < 0.4
        k, n = rng.choice([(256, 256), (256, 512), (512, 256), (256, 1024), (1024, 256),
                           (2048, 2048), (2048, 8192), (1024, 4096), (256, 128), (256, 96),
                           (320, 1280), (100, 300), (75, 257), (1001, 64),
                           (_log(rng, 32, 2048), _log(rng, 32, 2048))])
        act = rng.choice(["none", "relu", "silu", "gelu"])
        if train and dtype == "fp32" and act == "relu":
            act = "gelu"  # (one sign next to zero would decide about a whole value)
        rows = _log(rng, 1, 200000)
        cost = (12 if dtype == "fp32" else 3) if train else (4 if dtype == "fp32" else 1)
        while rows * k * n * cost > 2 ** 36 or rows * (k + n) * cost > 2 ** 27:
            rows -= -(-rows // 8)
        return _unnamed(_linear("", max(rows, 1), k, n, act, rng.random() < 0.5, dtype, train))
    if op == "norm":
        train = rng.random() < 0.6
        channels = rng.choice([256, 256, 512, 1024, 2048, 4096, 8192, 128, 64, 320, 100, 75, 1001,
                               _log(rng, 16, 4096)])
        sets, rows = rng.randint(1, 8), _log(rng, 1, 40000)
        limit = 2 ** 25 // (4 if train else 1)
        while sets * rows * channels > limit:
            rows -= -(-rows // 8)
        return _unnamed(_norm("", sets, rows, channels, rng.choice(["layer", "layer", "rms"]),
                              rng.choice(["none", "channels", "sets"]), rng.random() < 0.4,
                              rng.random() < 0.6, dtype, train))
    width = rng.choice([64, 100, 128, 256, 320, 512, 1000, 1024])
    layers = _log(rng, 1, 12) if width < 1000 else _log(rng, 1, 5)
    rows = rng.choice([0, 300, _log(rng, 1000, 32768)])
    return _unnamed(_adamw("", rows, width, layers, rng.choice([8, 32]), dtype,
                           rng.random() < 0.5, rng.choice([0.0, 1.0, 35.0])))


def _unnamed(case):
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------

def _linear_inputs(case, rand):
    m, k, n, dt = case["rows"], case["k"], case["n"], DTYPES[case["dtype"]]
    s = {"x": rand(m, k).to(dt), "weight": (rand(n, k) / k ** 0.5).to(dt),
         "bias": (0.2 * rand(n)).to(dt), "residual": rand(m, n).to(dt) if case["residual"] else None}
    if case["train"]:
        s["grad"] = rand(m, n).to(dt)
    return s


def _norm_inputs(case, rand):
    """The stream with a mean and a spread for each channel, the block's output smaller."""
    b, m, c, dt = case["sets"], case["rows"], case["channels"], DTYPES[case["dtype"]]
    s = {"x": (0.5 * rand(b, m, c) * (0.5 + rand(c).abs())).to(dt),
         "residual": (rand(b, m, c) * (0.5 + rand(c).abs()) + 0.5 * rand(c)).to(dt),
         "weight": (1 + 0.2 * rand(c)).to(dt),
         "bias": (0.2 * rand(c)).to(dt) if case["kind"] == "layer" else None,
         "gate": None, "block_weight": None, "block_bias": None}
    if case["gate"] != "none":
        s["gate"] = (0.5 + 0.3 * rand(*((b, c) if case["gate"] == "sets" else (c,)))).to(dt)
    if case["block_norm"]:
        s["block_weight"] = (1 + 0.2 * rand(c)).to(dt)
        if case["kind"] == "layer":
            s["block_bias"] = (0.2 * rand(c)).to(dt)
    if case["train"]:
        s["grad"] = rand(b, m, c).to(dt)
        if case["stream"]:
            s["grad_stream"] = rand(b, m, c).to(dt)
    return s


_NORM_LEAVES = ("x", "residual", "weight", "bias", "gate", "block_weight", "block_bias")


def _shapes(case):
    """An embedding table or none, then for each layer four square matrices with their
    biases, two matrices of four times the width, and two norms."""
    d = case["width"]
    layer = [(d, d), (d,)] * 4 + [(4 * d, d), (4 * d,), (d, 4 * d), (d,)] + [(d,)] * 4
    return ([(case["rows"], d)] if case["rows"] else []) + layer * case["layers"]


def _pieces(flat, shapes):
    """The tensors of those shapes in a flat buffer, each at a multiple of BLOCK values."""
    sizes = [math.prod(s) for s in shapes]
    parts = flat.split([-(-n // BLOCK) * BLOCK for n in sizes])
    return [p[:n].view(s) for p, n, s in zip(parts, sizes, shapes)]


def _adamw_inputs(case, rand, uniform):
    """The weights after some steps: gradients of a spread of 0.01, moments that fit them."""
    shapes = _shapes(case)
    total = sum(-(-math.prod(s) // BLOCK) * BLOCK for s in shapes)
    there = torch.zeros(total, device=DEV)  # (what lies between two tensors is zero and stays so)
    [t.fill_(1) for t in _pieces(there, shapes)]
    params = 0.06 * rand(total) * there
    grads = [(0.01 * rand(*s)).to(DTYPES[case["grads"]]) for s in shapes]
    if case["bits"] == 32:
        state = {"exp_avg": 0.003 * rand(total) * there,
                 "exp_avg_sq": 1e-4 * (0.3 + uniform(total)) * there}
    else:  # codes of three mantissa bits, an exponent for each block
        blocks = total // BLOCK
        state = {"exp_avg": (uniform(total) * 256 * there).to(torch.uint8),
                 "exp_avg_sq": ((216 + uniform(total) * 40) * there).to(torch.uint8),
                 "exp_avg_scale": torch.full((blocks,), 120, dtype=torch.uint8, device=DEV),
                 "exp_avg_sq_scale": torch.full((blocks,), 114, dtype=torch.uint8, device=DEV)}
    state["step"] = torch.full((1,), 100, dtype=torch.int64, device=DEV)
    state["seed"] = 1234567
    s = {"flat": params, "params": _pieces(params, shapes), "grads": grads, "state": state,
         "flat_copies": None, "copies": None, "norm": None}
    if case["copies"]:
        s["flat_copies"] = params.to(torch.bfloat16)
        s["copies"] = _pieces(s["flat_copies"], shapes)
    if case["max_norm"]:
        s["norm"] = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt().float()
    return s


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def rand(*size):
        return torch.randn(*size, device=DEV, generator=gen)

    def uniform(*size):
        return torch.rand(*size, device=DEV, generator=gen)

    if case["op"] == "adamw":
        s = _adamw_inputs(case, rand, uniform)
    else:
        s = (_linear_inputs if case["op"] == "linear" else _norm_inputs)(case, rand)
        if case["train"]:
            [s[k].requires_grad_() for k in _NORM_LEAVES if s.get(k) is not None]
    return dict(s, case=case)


# ---------------------------------------------------------------------------------------
# One pass: the library's calls, or the plain form
# ---------------------------------------------------------------------------------------

def run(state):
    """The outputs; for a training step also the gradients."""
    case = state["case"]
    form = {"linear": (_linear_plain, _linear_own), "norm": (_norm_plain, _norm_own),
            "adamw": (_adamw_plain, _adamw_own)}[case["op"]]
    return form[1](state, case) if own else form[0](state, case)


def _act(case):
    return None if case["act"] == "none" else case["act"]


def _leaves(s, names):
    return [s[k] for k in names if s.get(k) is not None]


def _linear_own(s, case):
    from msda_opt2 import linear_act
    args = (s["x"], s["weight"], s["bias"], _act(case), s["residual"])
    if not case["train"]:
        with torch.no_grad():
            return [linear_act(*args)]
    y = linear_act(*args)
    leaves = _leaves(s, ("x", "weight", "bias", "residual"))
    return [y.detach(), *torch.autograd.grad(y, leaves, s["grad"])]


def _norm_own(s, case):
    from msda_opt2 import residual_norm
    block = (s["block_weight"], s["block_bias"]) if case["block_norm"] else None
    kwargs = {"gate": s["gate"], "scale": 0.7, "block_norm": block, "kind": case["kind"],
              "eps": EPS, "with_stream": case["stream"]}
    args = (s["x"], s["residual"], s["weight"], s["bias"])
    if not case["train"]:
        with torch.no_grad():
            out = residual_norm(*args, **kwargs)
        return list(out) if case["stream"] else [out]
    out = residual_norm(*args, **kwargs)
    out = out if case["stream"] else (out,)
    grads = (s["grad"], s["grad_stream"]) if case["stream"] else (s["grad"],)
    return [*(o.detach() for o in out), *torch.autograd.grad(out, _leaves(s, _NORM_LEAVES), grads)]


def _adamw_own(s, case):
    from modulated_deform_conv import adamw_moments, adamw_step_
    adamw_step_(s["params"], s["grads"], s["state"], lr=LR, betas=BETAS, eps=ADAM_EPS,
                weight_decay=DECAY, norm=s["norm"], max_norm=case["max_norm"] or None,
                copies=s["copies"])
    dtype = torch.float32 if case["bits"] == 32 else torch.bfloat16  # (exact for 8 bits)
    return [s["flat"], *adamw_moments(s["state"], dtype), s["state"]["step"], s["flat_copies"]]


@torch.no_grad()
def _linear_plain(s, case):
    x, w, dt = s["x"].float(), s["weight"].float(), s["x"].dtype
    z = x @ w.t() + s["bias"].float()
    slope = None
    if case["act"] == "relu":
        y = z.clamp(min=0)
        if case["train"]:  # next to zero the sign of z takes 64 bits
            slope = (x.double() @ w.double().t() + s["bias"].double() > 0).float()
    elif case["act"] == "silu":
        sig = 1 / (1 + torch.exp(-z))
        y = z * sig
        slope = sig * (1 + z * (1 - sig)) if case["train"] else None
    elif case["act"] == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        y = z * cdf
        if case["train"]:
            slope = cdf + z * torch.exp(-0.5 * z * z) * (0.5 / math.pi) ** 0.5
    else:
        y = z
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if not case["train"]:
        return [y.to(dt)]
    g = s["grad"].float()
    gz = g if slope is None else g * slope
    grads = [(gz @ w).to(dt), (gz.t() @ x).to(dt), gz.sum(0).to(dt)]
    return [y.to(dt), *grads] + ([s["grad"].clone()] if s["residual"] is not None else [])


def _normed(v, kind):
    """v over its spread, and 1 over the spread."""
    d = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    rstd = torch.rsqrt(d.square().mean(-1, keepdim=True) + EPS)
    return d * rstd, rstd


def _norm_back(g, vh, rstd, kind):
    """The gradient of v for the gradient g of its normed value vh."""
    g2 = g - vh * (g * vh).mean(-1, keepdim=True)
    return rstd * (g2 - g.mean(-1, keepdim=True) if kind == "layer" else g2)


@torch.no_grad()
def _norm_plain(s, case):
    dt, kind = s["x"].dtype, case["kind"]
    f = {k: s[k].float() if s[k] is not None else None for k in _NORM_LEAVES}
    gate = 0.7
    if s["gate"] is not None:
        gate = 0.7 * (f["gate"].unsqueeze(1) if case["gate"] == "sets" else f["gate"])
    p = f["x"]
    if case["block_norm"]:
        ph, prstd = _normed(p, kind)
        p = ph * f["block_weight"]
        p = p if f["block_bias"] is None else p + f["block_bias"]
    h = f["residual"] + gate * p
    hh, rstd = _normed(h, kind)
    y = hh * f["weight"]
    y = y if f["bias"] is None else y + f["bias"]
    out = [y.to(dt), h.to(dt)] if case["stream"] else [y.to(dt)]
    if not case["train"]:
        return out
    g = s["grad"].float()
    gh = _norm_back(g * f["weight"], hh, rstd, kind)
    gh = gh + s["grad_stream"].float() if case["stream"] else gh
    gp = gate * gh
    rows = (0, 1)
    gx = _norm_back(gp * f["block_weight"], ph, prstd, kind) if case["block_norm"] else gp
    grads = {"x": gx, "residual": gh, "weight": (g * hh).sum(rows),
             "bias": g.sum(rows), "gate": 0.7 * (gh * p).sum(1 if case["gate"] == "sets" else rows),
             "block_weight": (gp * ph).sum(rows) if case["block_norm"] else None,
             "block_bias": gp.sum(rows)}
    return out + [grads[k].to(dt) for k in _NORM_LEAVES if s[k] is not None]


# The 8-bit moments. exp_avg: sign, 4 exponent and 3 mantissa bits; exp_avg_sq: 5 and 3; the largest
# exponent stands for the block's scale (a biased exponent of fp32), code 0 (and 128) for zero. A value
# is rounded to three mantissa bits by adding 20 random bits below them: 16 from a mixing function of
# its place in the flat buffer, the step and the seed, and a half.

def _mul32(x, c):
    """The low 32 bits of x * c, for x below 2^32 in int64."""
    return ((x & 0xffff) * c + (((x >> 16) * c & 0xffff) << 16)) & 0xffffffff


def _mix(x):
    x = _mul32(x & 0xffffffff, 0x9E3779B1)
    x = _mul32(x ^ (x >> 15), 0xB504F333)
    x = _mul32(x ^ (x >> 13), 0x9E3779B1)
    return x ^ (x >> 16)


def _random(total, step, seed):
    """32 random bits for each place: the high half for exp_avg, the low one for exp_avg_sq."""
    place = torch.arange(total, device=DEV)
    low, high = seed & 0xffffffff, seed >> 32 & 0xffffffff
    key = _mix(_mix(_mix(_mix(torch.full_like(step, low)) + high) + (step & 0xffffffff))
               + (step >> 32))
    return _mix(place + _mix(key + (place >> 32)))


def _coded(v, rand16, top):
    """(codes, scales) of values v >= 0 (fp32): exponents up to `top`, three mantissa bits."""
    bits = v.view(torch.int32).long()
    scale = ((bits.view(-1, BLOCK).amax(1) + 0xfffff) >> 23).clamp(top + 1, 255)
    q = ((bits + rand16 * 16 + 8) >> 20).view(-1, BLOCK) - ((scale - top) << 3).unsqueeze(1)
    q = q.clamp(max=top * 8 + 7)
    least = (v > 0).view(-1, BLOCK) * 8 if top == 31 else 0  # a second moment never vanishes
    return torch.where(q < 8, least, q).flatten().to(torch.uint8), scale.to(torch.uint8)


def _decoded(codes, scale, top):
    q = codes.long().view(-1, BLOCK)
    size = q & (top * 8 + 7)
    bits = (size + ((scale.long() - top) << 3).unsqueeze(1)) << 20
    v = torch.where(size < 8, 0, bits).int().view(torch.float32).flatten()
    return torch.where(codes >= 128, -v, v) if top == 15 else v


def _flat_grads(s, total, dtype):
    flat = torch.zeros(total, dtype=dtype, device=DEV)
    [p.copy_(g) for p, g in zip(_pieces(flat, [g.shape for g in s["grads"]]), s["grads"])]
    return flat


@torch.no_grad()
def _adamw_plain(s, case):
    st, p = s["state"], s["flat"]
    total = p.numel()
    st["step"] += 1
    (b1, b2), t = BETAS, st["step"].double()
    size = (LR / (1 - b1 ** t)).float()
    root = (1 / torch.sqrt(1 - b2 ** t)).float()
    g = _flat_grads(s, total, torch.float32)
    if case["max_norm"]:
        g = g * (case["max_norm"] / (s["norm"] + 1e-6)).clamp(max=1)
    if case["bits"] == 32:
        m, v = st["exp_avg"], st["exp_avg_sq"]
    else:
        m = _decoded(st["exp_avg"], st["exp_avg_scale"], 15)
        v = _decoded(st["exp_avg_sq"], st["exp_avg_sq_scale"], 31)
    m = ((m * b1).double() + g.double() * (1 - b1)).float()  # (next to a rounding's border)
    v = ((v * b2).double() + g.square().double() * (1 - b2)).float()
    p.copy_(p * (1 - LR * DECAY) - size * m / (torch.sqrt(v) * root + ADAM_EPS))
    if case["bits"] == 32:
        st["exp_avg"].copy_(m)
        st["exp_avg_sq"].copy_(v)
    else:
        rand = _random(total, st["step"], st["seed"])
        codes, scale = _coded(m.abs(), rand >> 16, 15)
        codes = codes + (m < 0).to(torch.uint8) * 128
        st["exp_avg"].copy_(codes)
        st["exp_avg_scale"].copy_(scale)
        m = _decoded(codes, scale, 15).to(torch.bfloat16)
        codes, scale = _coded(v, rand & 0xffff, 31)
        st["exp_avg_sq"].copy_(codes)
        st["exp_avg_sq_scale"].copy_(scale)
        v = _decoded(codes, scale, 31).to(torch.bfloat16)
    if s["copies"] is not None:
        s["flat_copies"].copy_(p)
    return [p, m, v, st["step"], s["flat_copies"]]


# ---------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------

def work(case):
    if case["op"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case))
        moments = 16 if case["bits"] == 32 else 4 + 4 / BLOCK + 4  # (8 bits: also given as bf16)
        grads = 4 if case["grads"] == "fp32" else 2
        return {"bytes": n * (8 + grads + moments + (2 if case["copies"] else 0)),
                "flops": 14.0 * n}
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        ahead = m * k + n * k + n + m * n * (2 if case["residual"] else 1)
        if not case["train"]:
            return {"bytes": size * ahead, "flops": 2.0 * m * n * k}
        # backward: the output's gradient, x and W read, three gradients written
        return {"bytes": size * (ahead + m * n + 2 * m * k + 2 * n * k + n),
                "flops": 6.0 * m * n * k}
    n = case["sets"] * case["rows"] * case["channels"]
    ahead = 4 if case["stream"] else 3
    if not case["train"]:
        return {"bytes": size * ahead * n, "flops": 10.0 * n}
    # backward: the outputs' gradients, the stream (and the block's output) read, two written
    back = 4 + case["stream"] + (case["gate"] != "none" or case["block_norm"])
    return {"bytes": size * (ahead + back) * n, "flops": 30.0 * n}


# ---------------------------------------------------------------------------------------
# The same in 64 bits
# ---------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _adamw_exact(s, case)
    d = {k: v.detach().double().requires_grad_(case["train"])
         for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["op"] == "linear":
        z = F.linear(d["x"], d["weight"], d["bias"])
        y = {"relu": F.relu, "silu": F.silu, "gelu": F.gelu, "none": lambda t: t}[case["act"]](z)
        out = [y + d["residual"] if case["residual"] else y]
        names = ("x", "weight", "bias", "residual")
    else:
        def norm(v, w, b):
            if case["kind"] == "layer":
                return F.layer_norm(v, v.shape[-1:], w, b, EPS)
            return F.rms_norm(v, v.shape[-1:], w, EPS)

        p = d["x"]
        if case["block_norm"]:
            p = norm(p, d["block_weight"], d.get("block_bias"))
        if case["gate"] != "none":
            p = p * (d["gate"][:, None] if case["gate"] == "sets" else d["gate"])
        h = d["residual"] + 0.7 * p
        y = norm(h, d["weight"], d.get("bias"))
        out = [y, h] if case["stream"] else [y]
        names = _NORM_LEAVES
    if not case["train"]:
        return out
    grads = [d["grad"], d["grad_stream"]] if len(out) == 2 else [d["grad"]]
    found = torch.autograd.grad(out, [d[k] for k in names if k in d], [g.detach() for g in grads])
    return [*(o.detach() for o in out), *found]


def _adamw_exact(s, case):
    st = s["state"]
    t = st["step"].item() + 1
    m, v = st["exp_avg"], st["exp_avg_sq"]
    if case["bits"] == 8:
        def value(codes, scale, top):
            q = codes.view(-1, BLOCK).double()
            sign = 1 - 2 * (q >= 128) if top == 15 else 1
            q = q % 128 if top == 15 else q
            e = torch.floor(q / 8)
            size = (1 + (q - 8 * e) / 8) * torch.exp2(e - top + scale.double()[:, None] - 127)
            return (sign * size * (q >= 8)).flatten()

        m = value(m, st["exp_avg_scale"], 15)
        v = value(v, st["exp_avg_sq_scale"], 31)
    g = _flat_grads(s, s["flat"].numel(), torch.float64)
    if case["max_norm"]:
        g *= min(1.0, case["max_norm"] / (s["norm"].item() + 1e-6))
    m = BETAS[0] * m.double() + (1 - BETAS[0]) * g
    v = BETAS[1] * v.double() + (1 - BETAS[1]) * g * g
    up = (m / (1 - BETAS[0] ** t)) / (torch.sqrt(v / (1 - BETAS[1] ** t)) + ADAM_EPS)
    p = (1 - LR * DECAY) * s["flat"].double() - LR * up
    if case["bits"] == 8:  # what is kept is a random neighbour: nothing to compare with
        m = v = None
    copies = p if case["copies"] else None
    return [p, m, v, None, copies]
