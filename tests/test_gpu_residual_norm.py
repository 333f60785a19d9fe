"""The norms between two blocks (residual_norm_fwd.hip, residual_norm_bwd.hip) against the formulas in
64 bits.

Bounds, with u = 2^-24 and e the half step of the type that is written (finfo.eps / 2). A sum over C
channels is at most D = C / (threads of a row) + 10 additions deep; k = D u of the sum of magnitudes.
  N(v)  mean off by k mean|v|, v - mean by u more; rstd by (k + 4 u) + what the mean's error gives in
        second order; three roundings behind: with dv the error of v itself,
        dn = |w| rstd (2 dv + k mean|v| + 2 u |v - mean|) + (k + 8 u) |w n| + u |b|
  h     dp scale |gate| + 3 u (|residual| + |scale gate p|)
  y     dn at v = h; then e |y|
  the backward computes the same h again
  sums over the rows: D of at most 64 + rows / 16 additions, (D + 8) u of the sum of magnitudes and
        the terms' own errors
  gh, gx: the terms' errors times |rstd| and 8 u of their magnitudes, then e"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
NAMES = ("x", "residual", "weight", "bias", "gate", "block_weight", "block_bias")


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _inputs(shape, dtype, seed, gate=None, block=True, ptype=None, mean=0.5, affine=True, residual=True):
    g = torch.Generator().manual_seed(seed)
    c = shape[-1]

    def rand(*s):
        return torch.randn(*s, generator=g)

    t = {"x": rand(*shape) * (0.3 + torch.rand(c, generator=g)),
         "residual": rand(*shape) + mean if residual else None,
         "weight": 1 + 0.3 * rand(c) if affine else None, "bias": 0.3 * rand(c) if affine else None,
         "gate": None if gate is None else 0.5 + 0.4 * rand(*((c,) if gate == "channels" else (shape[0], c))),
         "block_weight": 1 + 0.3 * rand(c) if block and affine else None,
         "block_bias": 0.3 * rand(c) if block and affine else None}
    grads = rand(*shape).to(dtype), rand(*shape).to(dtype)
    types = {n: dtype if n in ("x", "residual") else ptype or dtype for n in NAMES}
    return {n: None if v is None else v.to(types[n]) for n, v in t.items()}, grads


class _Norm:
    """N(v) with v's error, and its gradient."""

    def __init__(self, v, dv, w, b, kind, eps, k):
        c = v.shape[-1]
        self.w = torch.ones(c, dtype=torch.float64) if w is None else w
        b = torch.zeros(c, dtype=torch.float64) if b is None else b
        self.kind = kind
        mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
        d = v - mean
        self.rstd = 1 / torch.sqrt(d.square().mean(-1, keepdim=True) + eps)
        self.n = d * self.rstd
        dmean = k * v.abs().mean(-1, keepdim=True) if kind == "layer" else 0
        # (an error of the mean enters the variance in second order alone; dv's own is averaged over n)
        self.drel = k + 8 * U + 2 * self.rstd * (dv * self.n.abs()).mean(-1, keepdim=True) \
            + (dmean * self.rstd) ** 2
        self.dn = self.rstd * (dv + dv.mean(-1, keepdim=True) + dmean + 2 * U * d.abs()) + self.drel * self.n.abs()
        self.y = self.n * self.w + b
        self.dy = self.w.abs() * self.dn + 2 * U * (self.n * self.w).abs() + U * b.abs()

    def back(self, g, dg, k):
        """The gradient of v for that of N(v), with errors; also of w and b for each row."""
        t, dt = g * self.w, (dg + U * g.abs()) * self.w.abs()
        c1 = t.mean(-1, keepdim=True) if self.kind == "layer" else 0 * self.rstd
        dc1 = (dt + k * t.abs()).mean(-1, keepdim=True) if self.kind == "layer" else 0
        c2 = (t * self.n).mean(-1, keepdim=True)
        dc2 = (dt * self.n.abs() + t.abs() * self.dn + k * (t * self.n).abs()).mean(-1, keepdim=True)
        out = self.rstd * (t - c1 - self.n * c2)
        err = self.rstd * (dt + dc1 + self.n.abs() * dc2 + self.dn * c2.abs()
                           + (8 * U + self.drel) * (t.abs() + c1.abs() + (self.n * c2).abs()))
        return out, err


class Reference:
    def __init__(self, t, gy, gs, scale, block, kind, eps):
        d = {n: None if v is None else v.double() for n, v in t.items()}
        c = t["x"].shape[-1]
        k = (c / 16 + 14) * U if c > 16 else 24 * U
        k = min(k, (8 + 24) * U) if c <= 8192 else (c / 256 + 20) * U
        lead = [1] * (t["x"].dim() - 2)
        gate = torch.ones(c, dtype=torch.float64) if d["gate"] is None else d["gate"]
        gate = gate.view(-1, *lead, c) if gate.dim() > 1 else gate
        res = torch.zeros_like(d["x"]) if d["residual"] is None else d["residual"]
        zero = torch.zeros_like(d["x"])
        p, dp = d["x"], zero
        if block:
            bn = _Norm(d["x"], zero, d["block_weight"], d["block_bias"], kind, eps, k)
            p, dp = bn.y, bn.dy
        up = scale * gate * p
        self.h = res + up
        self.h_err = abs(scale) * gate.abs() * dp + 3 * U * (res.abs() + up.abs())
        n = _Norm(self.h, self.h_err, d["weight"], d["bias"], kind, eps, k)
        self.y, self.y_err = n.y, n.dy
        g = gy.double()
        gh, gh_err = n.back(g, zero, k)
        if gs is not None:
            gh, gh_err = gh + gs.double(), gh_err + U * (gh + gs.double()).abs()
        rows = self.h.numel() // c
        deep = (rows / 16 + 72) * U
        gp, gp_err = scale * gate * gh, abs(scale) * gate.abs() * (gh_err + 3 * U * gh.abs())

        def summed(v, dv, to):
            total = (deep * v.abs() + dv)
            if to is not None and to.dim() > 1:
                flat = (to.shape[0], -1, c)
                return v.reshape(flat).sum(1), total.reshape(flat).sum(1)
            return v.reshape(-1, c).sum(0), total.reshape(-1, c).sum(0)

        self.grads = {"residual": (gh, gh_err),
                      "weight": summed(g * n.n, g.abs() * n.dn, None), "bias": summed(g, zero, None),
                      "gate": summed(scale * gh * p, abs(scale) * (gh_err * p.abs() + gh.abs() * dp), d["gate"]),
                      "x": (gp, gp_err)}
        if block:
            self.grads["x"] = bn.back(gp, gp_err, k)
            self.grads["block_weight"] = summed(gp * bn.n, gp_err * bn.n.abs() + gp.abs() * bn.dn, None)
            self.grads["block_bias"] = summed(gp, gp_err, None)


def _near(got, ref, err, what):
    got = got.detach().cpu()
    half = _half_step(got.dtype)
    bound = err + half * (ref.abs() + err) + torch.finfo(got.dtype).smallest_normal * half
    off = (got.double().reshape(ref.shape) - ref).abs()
    assert (off <= bound).all(), f"{what}: worst {(off / bound).max().item():.3f} of the bound"


def _run(t, gy, gs, scale, block, kind, eps, leaves=None):
    from msda_opt2 import residual_norm
    leaves = leaves or {n: None if v is None else v.to(DEV).requires_grad_() for n, v in t.items()}
    out = residual_norm(leaves["x"], leaves["residual"], leaves["weight"], leaves["bias"], leaves["gate"], scale,
                        (leaves["block_weight"], leaves["block_bias"]) if block else None, kind, eps,
                        with_stream=gs is not None)
    out = out if gs is not None else (out,)
    grads = torch.autograd.grad(out, [v for v in leaves.values() if v is not None],
                                [g.to(DEV) for g in (gy, gs) if g is not None])
    return out, dict(zip([n for n, v in leaves.items() if v is not None], grads))


def _check(t, grads, scale=1.0, block=True, kind="layer", eps=1e-5, stream=True):
    gy, gs = grads if stream else (grads[0], None)
    out, found = _run(t, gy, gs, scale, block, kind, eps)
    r = Reference(t, gy, gs, scale, block, kind, eps)
    assert out[0].shape == t["x"].shape and out[0].dtype == t["x"].dtype
    _near(out[0], r.y, r.y_err, "y")
    if stream:
        _near(out[1], r.h, r.h_err, "stream")
    for name, g in found.items():
        assert g.dtype == t[name].dtype and g.shape == t[name].shape
        _near(g, *r.grads[name], f"gradient of {name}")
    return out, found


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("gate,block", [(None, False), ("channels", False), ("sets", False), (None, True),
                                        ("channels", True), ("sets", True)],
                         ids=["plain", "channels", "sets", "block", "block-channels", "block-sets"])
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 1, 256), (3, 5, 8), (2, 37, 75), (2, 300, 256), (3, 33, 100),
                                   (1, 70, 1001), (2, 9, 2048), (1, 3, 4096)], ids=str)
def test_residual_norm(shape, gate, block, dtype, kind):
    t, grads = _inputs(shape, TYPES[dtype], shape[1] + shape[2], gate, block)
    _check(t, grads, 0.7, block, kind)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(2, 3, 8192), (1, 2, 16384), (1, 3, 16400), (2, 2, 5000), (1, 2, 3333),
                                   (1, 1, 40000)], ids=str)
def test_long_rows(shape, dtype):
    t, grads = _inputs(shape, TYPES[dtype], shape[2], "sets", True)
    _check(t, grads, 1.0, True, "layer")


@pytest.mark.parametrize("stream", [True, False])
@pytest.mark.parametrize("scale", [1.0, 0.25])
def test_plain_residual(stream, scale):
    """Attention output plus residual, then the norm; with and without the stream's own gradient."""
    for residual in (True, False):
        t, grads = _inputs((4, 77, 256), torch.float32, 3, None, False, residual=residual)
        _check(t, grads, scale, False, stream=stream)


def test_without_parameters():
    for block in (False, True):
        t, grads = _inputs((2, 40, 96), torch.bfloat16, 4, None, block, affine=False)
        _check(t, grads, 1.0, block)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_fp32_parameters(dtype):
    t, grads = _inputs((2, 60, 128), TYPES[dtype], 5, "sets", True, torch.float32)
    _check(t, grads, 0.5)
    t["gate"] = t["gate"].to(TYPES[dtype])
    _check(t, grads, 0.5)


@pytest.mark.parametrize("sets,rows", [(1500, 1), (2000, 3), (1, 9000), (7, 1)])
def test_numbers_of_sets(sets, rows):
    t, grads = _inputs((sets, rows, 64), torch.float32, sets, "sets", True)
    _check(t, grads, 1.0)


def test_gate_for_each_row_and_with_ones_between():
    from msda_opt2 import residual_norm
    t, grads = _inputs((50, 64), torch.float32, 8, "sets", False)
    _check(t, grads, 1.0, False)
    t, _ = _inputs((3, 4, 5, 32), torch.float32, 9, "sets", False)
    x, r, gate = t["x"].to(DEV), t["residual"].to(DEV), t["gate"].to(DEV)
    a = residual_norm(x, r, gate=gate)
    b = residual_norm(x, r, gate=gate.view(3, 1, 1, 32))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_far_mean():
    """A mean of 1,000 spreads, and rows of one value."""
    t, grads = _inputs((2, 31, 256), torch.float32, 10, None, False, mean=1000.0)
    _check(t, grads)
    t["x"].zero_()
    t["residual"][1] = 3.0
    t["residual"][0] = 0.0
    out, _ = _check(t, grads)
    assert torch.equal(out[0][1].cpu(), t["bias"].expand(31, 256))


def test_non_finite_rows_stay_in_their_rows():
    from msda_opt2 import residual_norm
    t, _ = _inputs((1, 40, 256), torch.bfloat16, 11, "channels", True)
    good = residual_norm(*(t[n].to(DEV) for n in ("x", "residual", "weight", "bias", "gate")))
    for bad in (float("inf"), float("-inf"), float("nan")):
        x = t["x"].clone()
        x[0, 7, 100] = bad
        y, h = residual_norm(x.to(DEV), *(t[n].to(DEV) for n in ("residual", "weight", "bias", "gate")))
        rest = torch.arange(40) != 7
        assert torch.equal(y[0, rest.to(DEV)], good[0][0, rest.to(DEV)])
        assert y[0, 7].isnan().any() and not h[0, 7].isfinite().all()


def test_empty():
    from msda_opt2 import residual_norm
    x = torch.zeros(0, 5, 32, device=DEV, requires_grad=True)
    w = torch.ones(32, device=DEV, requires_grad=True)
    y, h = residual_norm(x, x.detach(), w)
    gx, gw = torch.autograd.grad([y, h], [x, w], [torch.zeros_like(y), torch.zeros_like(h)])
    assert y.shape == h.shape == gx.shape == x.shape and torch.equal(gw, torch.zeros_like(w))


def test_one_output_alone():
    """Only the stream's gradient, only y's, none for some of the inputs."""
    from msda_opt2 import residual_norm
    t, (gy, gs) = _inputs((2, 20, 128), torch.float32, 12, "sets", True)
    leaves = {n: v.to(DEV).requires_grad_() for n, v in t.items()}
    block = (leaves["block_weight"], leaves["block_bias"])
    y, h = residual_norm(leaves["x"], leaves["residual"], leaves["weight"], leaves["bias"], leaves["gate"], 0.5, block)
    r = Reference(t, torch.zeros_like(gy), gs, 0.5, True, "layer", 1e-5)
    for name in ("x", "residual", "gate", "block_bias"):
        g, = torch.autograd.grad(h, leaves[name], gs.to(DEV), retain_graph=True)
        _near(g, *r.grads[name], name)
    r = Reference(t, gy, None, 0.5, True, "layer", 1e-5)
    for name in NAMES:
        g, = torch.autograd.grad(y, leaves[name], gy.to(DEV), retain_graph=True)
        _near(g, *r.grads[name], name)


def test_views_and_strides():
    """Inputs that are not contiguous or not on 16 bytes, expanded gradients."""
    from msda_opt2 import residual_norm
    t, _ = _inputs((6, 10, 64), torch.bfloat16, 13, None, False)
    x = t["x"].to(DEV).requires_grad_()
    base = torch.randn(6 * 10 * 64 + 3, device=DEV).bfloat16()
    res = base[3:].view(6, 10, 64)
    y = residual_norm(x.transpose(0, 1), res.transpose(0, 1), t["weight"].to(DEV), with_stream=False)
    want = residual_norm(x.transpose(0, 1).contiguous(), res.transpose(0, 1).contiguous(), t["weight"].to(DEV),
                         with_stream=False)
    assert torch.equal(y, want)
    y.sum().backward()  # an expanded gradient
    assert x.grad.isfinite().all()


def test_differences():
    """The gradients against differences of the operator itself, along one direction, fp32: the
    central difference of step s is off by s^2 (third derivatives, below 40 here) and by 2^-24 * 2 / s
    of the sum's magnitude."""
    from msda_opt2 import residual_norm
    t, (gy, gs) = _inputs((2, 6, 64), torch.float32, 14, "sets", True)
    leaves = {n: v.to(DEV).requires_grad_() for n, v in t.items()}

    def value(of):
        y, h = residual_norm(of["x"], of["residual"], of["weight"], of["bias"], of["gate"], 0.6,
                             (of["block_weight"], of["block_bias"]))
        return (y.double() * gy.to(DEV)).sum() + (h.double() * gs.to(DEV)).sum(), (y * gy.to(DEV)).abs().sum().item()

    total, size = value(leaves)
    grads = dict(zip(leaves, torch.autograd.grad(total, list(leaves.values()))))
    gen = torch.Generator().manual_seed(15)
    for name in NAMES:
        step = 2.0 ** -7
        way = torch.randn(t[name].shape, generator=gen).to(DEV)
        way = way / way.norm()
        with torch.no_grad():
            ends = [value(dict(leaves, **{name: leaves[name] + k * step * way}))[0].item() for k in (1, -1)]
        slope = (grads[name].double() * way).sum().item()
        assert abs((ends[0] - ends[1]) / (2 * step) - slope) <= 40 * step ** 2 + 4 * U * size / step, name


def test_same_on_every_run_and_captured():
    """Forward and backward captured, replayed with new inputs between eager ones."""
    from msda_opt2 import residual_norm
    t, grads = _inputs((3, 500, 256), torch.bfloat16, 16, "sets", True)
    still = {n: v.to(DEV).requires_grad_() for n, v in t.items()}
    g = [v.to(DEV) for v in grads]

    def step(of):
        out = residual_norm(of["x"], of["residual"], of["weight"], of["bias"], of["gate"], 0.5,
                            (of["block_weight"], of["block_bias"]))
        return [*(o.detach() for o in out), *torch.autograd.grad(out, list(of.values()), g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(still)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(still)
    for k in range(4):
        new, _ = _inputs((3, 500, 256), torch.bfloat16, 20 + k, "sets", True)
        with torch.no_grad():
            for n, v in new.items():
                still[n].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        eager = step({n: v.to(DEV).requires_grad_() for n, v in new.items()})
        for a, b in zip(held, eager):
            assert torch.equal(a, b)


def test_two_streams():
    from msda_opt2 import residual_norm
    t, _ = _inputs((1, 4000, 256), torch.float32, 30, None, False)
    x, r = t["x"].to(DEV), t["residual"].to(DEV)
    want = residual_norm(x, r)[0]
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = []
    for _ in range(3):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                out.append(residual_norm(x, r)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in out)


def test_forward_mode_and_second_derivatives_are_refused():
    from msda_opt2 import residual_norm
    import torch.autograd.forward_ad as fwd
    x = torch.randn(4, 32, device=DEV, requires_grad=True)
    y, _ = residual_norm(x)
    g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    with fwd.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError):
        residual_norm(fwd.make_dual(x.detach(), torch.ones_like(x)))


def test_refusals_on_the_device():
    from msda_opt2 import residual_norm
    x = torch.zeros(4, 8, device=DEV)
    for kw, match in ((dict(residual=x.half()), "residual must be"), (dict(residual=x[:2]), "residual must be"),
                      (dict(residual=x.cpu()), "HIP"), (dict(weight=torch.ones(4, device=DEV)), "weight must be"),
                      (dict(weight=torch.ones(8)), "HIP"), (dict(gate=torch.ones(2, 8, device=DEV)), "gate must be"),
                      (dict(gate=torch.ones(8, device=DEV).half()), "gate has dtype"),
                      (dict(kind="batch"), "kind must be"), (dict(eps=-1.0), "eps"),
                      (dict(weight=torch.ones(8, device=DEV).double()), "weight has dtype")):
        with pytest.raises(RuntimeError, match=match):
            residual_norm(x, **kw)
    with pytest.raises(RuntimeError, match="one dtype"):
        residual_norm(x.half(), weight=torch.ones(8, device=DEV), bias=torch.ones(8, device=DEV).half())
    with pytest.raises(RuntimeError, match="not implemented"):
        residual_norm(x.double())
    with pytest.raises(RuntimeError, match="two dimensions"):
        residual_norm(x[0])
