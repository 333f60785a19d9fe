"""Projections with bias, activation and residual (linear.hip) against 64 bits.

Bounds, with u = 2^-24 and e the half step of the output's type (finfo.eps / 2). The matrix cores add
at least 4 terms (fp32) or 16 (16 bits, whose products are exact) at a time to a sum, so a sum of K terms
is D = K / 4 + 24 or K / 16 + 24 additions deep (sums in parts, over waves and of split operands are
shallower), with S the sum of the terms' magnitudes:
  z   (D + 4) u S + 2 u |z|
  y   slopes are below 1.13; SiLU and GELU evaluated to (16 + |z|) u |y|, GELU in 16 bits to
      1.5e-7 |z| more (the polynomial's own error is half of that); the residual's sum u; then e |y|
  gz  the slope is off by z's error times second derivatives below 0.8, evaluated to 32 u (1 + |z|)
      (16 bits: 3e-7 more) and kept with 2^-16 more in 16 bits; anything where ReLU's z is within its error of 0;
      then e |gz| where there is an activation
  gx, gW, gbias   sums of gz as above, over N, the rows, the rows; then e"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _inputs(rows, k, n, dtype, seed, residual=True, btype=None, bias=True, device="cpu"):
    g = torch.Generator(device=device).manual_seed(seed)

    def rand(*s):
        return torch.randn(*s, generator=g, device=device)

    return {"x": rand(rows, k).to(dtype), "weight": (rand(n, k) / k ** 0.5).to(dtype),
            "bias": rand(n).to(btype or dtype) if bias else None,
            "residual": rand(rows, n).to(dtype) if residual else None}, rand(rows, n).to(dtype)


class Reference:
    def __init__(self, t, gy, act):
        dtype = t["x"].dtype
        half, step = _half_step(dtype), 4 if dtype == torch.float32 else 16
        x, w = t["x"].double(), t["weight"].double()

        def deep(count):
            return (count / step + 28) * U

        self.z = x @ w.t() + (0 if t["bias"] is None else t["bias"].double())
        z_err = deep(x.shape[1]) * (x.abs() @ w.abs().t()) + 2 * U * self.z.abs()
        z, coarse = self.z, 0 if dtype == torch.float32 else 1.5e-7
        if act is None:
            y, s, s_err = z, torch.ones_like(z), torch.zeros_like(z)
        elif act == "relu":
            y, s = z.clamp(min=0), (z > 0).double()
            s_err = (z.abs() <= z_err + torch.finfo(dtype).smallest_normal).double()
        elif act == "silu":
            p = 1 / (1 + torch.exp(-z))
            y, s = z * p, p * (1 + z * (1 - p))
            s_err = 0.8 * z_err + 32 * U * (1 + z.abs())
        else:
            cdf = torch.special.ndtr(z)
            y, s = z * cdf, cdf + z * torch.exp(-z * z / 2) * (2 * torch.pi) ** -0.5
            s_err = 0.8 * z_err + 32 * U * (1 + z.abs()) + 2 * coarse
        if act in ("silu", "gelu") and dtype != torch.float32:
            s_err = s_err + 2.0 ** -16
        self.y_err = 1.13 * z_err + (0 if act in (None, "relu") else (16 + z.abs()) * U * y.abs()
                                     + coarse * z.abs())
        if t["residual"] is not None:
            y = y + t["residual"].double()
            self.y_err = self.y_err + U * y.abs()
        self.y = y
        g = gy.double()
        gz = g * s
        gz_err = torch.zeros_like(gz) if act is None else \
            g.abs() * s_err + half * (gz.abs() + g.abs() * s_err) + torch.finfo(dtype).smallest_normal * half
        self.gx, self.gx_err = gz @ w, gz_err @ w.abs() + deep(w.shape[0]) * (gz.abs() @ w.abs())
        self.gw = gz.t() @ x
        self.gw_err = gz_err.t() @ x.abs() + deep(x.shape[0]) * (gz.abs().t() @ x.abs())
        self.gb, self.gb_err = gz.sum(0), gz_err.sum(0) + (x.shape[0] / 16 + 80) * U * gz.abs().sum(0)


def _near(got, ref, err, what):
    got, half = got.detach(), _half_step(got.dtype)
    ref, err = ref.to(got.device), err.to(got.device)
    bound = err + half * (ref.abs() + err) + torch.finfo(got.dtype).smallest_normal * half
    off = (got.double().reshape(ref.shape) - ref).abs()
    assert (off <= bound).all(), f"{what}: worst {(off / bound).max().item():.3f} of the bound"


def _check(t, gy, act):
    from msda_opt2 import linear_act
    leaves = {n: None if v is None else v.to(DEV).requires_grad_() for n, v in t.items()}
    y = linear_act(leaves["x"], leaves["weight"], leaves["bias"], act, leaves["residual"])
    assert y.shape == gy.shape and y.dtype == gy.dtype
    names = [n for n, v in leaves.items() if v is not None]
    grads = dict(zip(names, torch.autograd.grad(y, [leaves[n] for n in names], gy.to(DEV))))
    r = Reference(t, gy, act)
    _near(y, r.y, r.y_err, "y")
    _near(grads["x"], r.gx, r.gx_err, "gradient of x")
    _near(grads["weight"], r.gw, r.gw_err, "gradient of weight")
    if "bias" in grads:
        assert grads["bias"].dtype == t["bias"].dtype
        _near(grads["bias"], r.gb, r.gb_err, "gradient of bias")
    if "residual" in grads:
        assert torch.equal(grads["residual"].cpu(), gy.cpu())
    with torch.no_grad():
        assert torch.equal(linear_act(leaves["x"], leaves["weight"], leaves["bias"], act, leaves["residual"]), y)
    return y, grads


SIZES = [(1, 1, 1), (3, 8, 8), (1, 256, 256), (4, 2048, 320), (17, 100, 75), (33, 32, 16), (64, 64, 64),
         (65, 40, 129), (127, 96, 128), (300, 256, 256), (257, 1001, 64), (130, 64, 1024), (1000, 512, 72),
         (640, 320, 256)]


@pytest.mark.parametrize("act,residual", [(None, True), ("relu", False), ("relu", True), ("silu", True),
                                          ("gelu", False)])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_linear(size, dtype, act, residual):
    _check(*_inputs(*size, TYPES[dtype], sum(size), residual), act)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows", [1, 2, 5, 15, 16, 17, 31, 32, 48, 63, 100, 255, 256, 300, 511, 513, 1024, 2049])
def test_numbers_of_rows(rows, dtype):
    _check(*_inputs(rows, 256, 512, TYPES[dtype], rows), "silu")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("k,n", [(32, 32), (64, 8), (72, 64), (96, 200), (128, 136), (160, 264), (192, 512), (224, 24),
                                 (8, 256), (16, 520), (36, 36), (104, 1000), (512, 4), (1024, 1023)])
def test_numbers_of_features(k, n, dtype):
    for rows in (6, 333):
        _check(*_inputs(rows, k, n, TYPES[dtype], k + n), "gelu")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_fp32_bias_and_none(dtype):
    for rows in (3, 400):
        t, gy = _inputs(rows, 256, 256, TYPES[dtype], 5, btype=torch.float32)
        _check(t, gy, "silu")
        t["bias"] = None
        _check(t, gy, None)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("size", [(40000, 256, 512), (5800, 512, 256), (2000, 1024, 4096), (9001, 256, 264),
                                  (20000, 100, 300)], ids=str)
def test_ordinary_sizes(size, dtype):
    """Against 64 bits on the device."""
    t, gy = _inputs(*size, TYPES[dtype], 7, device=DEV)
    _check(t, gy, "gelu")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("size", [(700, 1001, 77), (700, 1003, 1005), (500, 4, 1000), (1001, 516, 255), (600, 2048, 512),
                                  (2, 2048, 4096), (2000, 256, 4096), (5000, 256, 2048), (1000, 256, 12288),
                                  (3000, 512, 4104), (4000, 1024, 520)], ids=str)
def test_where_another_kernel_takes_over(size, dtype):
    """Odd rows; fp32 by tiles or cut into pieces; more columns than are streamed past."""
    t, gy = _inputs(*size, TYPES[dtype], 17, device=DEV)
    for act in (None, "silu"):
        _check(t, gy, act)


def test_shapes_of_x():
    from msda_opt2 import linear_act
    t, _ = _inputs(60, 64, 40, torch.float32, 9)
    x, w, b, r = (t[n].to(DEV) for n in ("x", "weight", "bias", "residual"))
    flat = linear_act(x, w, b, "relu", r)
    assert torch.equal(linear_act(x.view(3, 4, 5, 64), w, b, "relu", r.view(3, 4, 5, 40)), flat.view(3, 4, 5, 40))
    one = linear_act(x[0], w, b, "relu", r[0])
    assert one.shape == (40,) and (one - flat[0]).abs().max() <= 1e-5
    wide = torch.randn(60, 128, device=DEV)
    assert torch.equal(linear_act(wide[:, :64], w), linear_act(wide[:, :64].contiguous(), w))
    assert torch.equal(linear_act(x, w.t().contiguous().t()), linear_act(x, w))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_off_sixteen_bytes(dtype):
    """Tensors that begin off 16-byte boundaries, forward and backward."""
    from msda_opt2 import linear_act
    for rows in (5, 200):
        t, gy = _inputs(rows, 256, 264, TYPES[dtype], 11)

        def off(v):
            base = torch.empty(v.numel() + 1, dtype=v.dtype, device=DEV)
            base[1:] = v.flatten().to(DEV)
            return base[1:].view(v.shape)

        leaves = {n: off(v).requires_grad_() for n, v in t.items()}
        y = linear_act(leaves["x"], leaves["weight"], leaves["bias"], "silu", leaves["residual"])
        gx, gw, gb = torch.autograd.grad(y, [leaves[n] for n in ("x", "weight", "bias")], off(gy))
        r = Reference(t, gy, "silu")
        for got, ref, err in ((y, r.y, r.y_err), (gx, r.gx, r.gx_err), (gw, r.gw, r.gw_err), (gb, r.gb, r.gb_err)):
            _near(got, ref, err, "off")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows", [4, 500])
def test_non_finite_values_stay_in_their_rows(rows, dtype):
    """Inf and NaN in one row of x reach that row of y alone; one in a column of gy that column of gW."""
    from msda_opt2 import linear_act
    t, gy = _inputs(rows, 256, 264, TYPES[dtype], 12)
    w, b = t["weight"].to(DEV), t["bias"].to(DEV)
    good = linear_act(t["x"].to(DEV), w, b)
    for bad in (float("inf"), float("-inf"), float("nan")):
        x = t["x"].clone()
        x[2, 100] = bad
        y = linear_act(x.to(DEV), w, b)
        rest = torch.arange(rows, device=DEV) != 2
        # (an fp32 tile with a value that is not finite is computed another way: within its bound)
        r = Reference(dict(t, residual=None), gy, None)
        _near(y[rest], r.y[rest.cpu()], r.y_err[rest.cpu()], "other rows")
        if dtype != "fp32":
            assert torch.equal(y[rest], good[rest])
        assert not y[2].isfinite().any()
        leaf = w.clone().requires_grad_()
        g = gy.clone()
        g[1, 5] = bad
        gw, = torch.autograd.grad(linear_act(t["x"].to(DEV), leaf, b), leaf, g.to(DEV))
        keep = torch.arange(264) != 5
        assert gw[keep.to(DEV)].isfinite().all() and not gw[5].isfinite().any()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,features,residual", [(4, 264, False), (4, 264, True), (500, 264, False), (500, 264, True),
                                                    (4000, 256, False), (4000, 256, True), (500, 261, True)])
def test_relu_of_nan(rows, features, residual, dtype):
    """A NaN is what ReLU makes of it, and its gradient goes on as it came (as torch's does)."""
    from msda_opt2 import linear_act
    t, gy = _inputs(rows, 256, features, TYPES[dtype], 16)
    r = t["residual"].to(DEV) if residual else None
    x = t["x"].to(DEV)
    x[2, 100] = float("nan")
    leaf, w, b = x.requires_grad_(), t["weight"].to(DEV), t["bias"].to(DEV)
    y = linear_act(leaf, w, b, "relu", r)
    assert y[2].isnan().all()
    gx, = torch.autograd.grad(y, leaf, gy.to(DEV))
    plain, = torch.autograd.grad(linear_act(leaf, w, b, None, r), leaf, gy.to(DEV))
    assert torch.equal(gx[2], plain[2]) and not torch.equal(gx, plain)


@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("size", [(1, 1, 1), (1, 100, 300), (1, 256, 256), (3, 33, 1), (2, 1, 40), (7, 2048, 512), (15, 257, 1001),
                                  (16, 64, 64), (16, 1024, 1024)], ids=str)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_gradients_of_few_rows(size, dtype, act):
    """Up to 16 rows of 16 bits: gz is not rounded, so the gradients have one rounding. The slope is off by its
    half step 2^-16, exp's and the formula's roundings (below 32 u of 1.13) and what z's error does to it (its
    derivative is below 0.8); each product adds its own and its sum's."""
    rows, k, n = size
    t, gy = _inputs(rows, k, n, TYPES[dtype], sum(size) + 1, False)
    _, grads = _check(t, gy, act)
    if act == "relu":  # (next to 0 the sign of z is not certain)
        return
    u, d = 2.0 ** -24, {m: v.double() for m, v in t.items() if v is not None}
    z = (d["x"] @ d["weight"].t() + d["bias"]).requires_grad_()
    gz, = torch.autograd.grad(getattr(torch.nn.functional, act)(z), z, gy.double())
    z_err = (k / 4 + 28) * u * (d["x"].abs() @ d["weight"].abs().t() + d["bias"].abs())
    gz_err = gy.double().abs() * (2.0 ** -16 + 32 * 1.13 * u + 0.8 * z_err) + u * gz.abs()
    for name, ref, err, mag, terms in (
            ("x", gz @ d["weight"], gz_err @ d["weight"].abs(), gz.abs() @ d["weight"].abs(), n),
            ("weight", gz.t() @ d["x"], gz_err.t() @ d["x"].abs(), gz.abs().t() @ d["x"].abs(), rows)):
        err = err + (terms + 28) * u * (mag + err)
        half = _half_step(TYPES[dtype])
        bound = err + half * (ref.abs() + err) + torch.finfo(TYPES[dtype]).smallest_normal * half
        assert ((grads[name].cpu().double() - ref).abs() <= bound).all(), name


def test_empty():
    from msda_opt2 import linear_act
    x = torch.zeros(0, 5, 32, device=DEV, requires_grad=True)
    w = torch.ones(16, 32, device=DEV, requires_grad=True)
    b = torch.ones(16, device=DEV, requires_grad=True)
    y = linear_act(x, w, b, "silu")
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.zeros_like(y))
    assert y.shape == (0, 5, 16) and gx.shape == x.shape
    assert torch.equal(gw, torch.zeros_like(w)) and torch.equal(gb, torch.zeros_like(b))


@pytest.mark.parametrize("act", [None, "gelu"])
def test_some_gradients(act):
    """One input's gradient alone is that of all together."""
    from msda_opt2 import linear_act
    t, gy = _inputs(333, 256, 128, torch.bfloat16, 13)
    leaves = {n: v.to(DEV).requires_grad_() for n, v in t.items()}
    y = linear_act(leaves["x"], leaves["weight"], leaves["bias"], act, leaves["residual"])
    names = list(leaves)
    both = torch.autograd.grad(y, list(leaves.values()), gy.to(DEV), retain_graph=True)
    for n, want in zip(names, both):
        rest = {m: v if m == n else v.detach() for m, v in leaves.items()}
        y = linear_act(rest["x"], rest["weight"], rest["bias"], act, rest["residual"])
        got, = torch.autograd.grad(y, leaves[n], gy.to(DEV))
        assert torch.equal(got, want), n


def test_differences():
    """The gradients against differences of the operator itself along one direction, fp32: a central
    difference of step s is off by s^2 / 6 of the third derivative (below 3 here along a unit direction
    and 20 in all) and by 2 * 2^-24 / s of the sum's magnitude."""
    from msda_opt2 import linear_act
    t, gy = _inputs(12, 64, 48, torch.float32, 14)
    leaves = {n: v.to(DEV).requires_grad_() for n, v in t.items()}
    gen = torch.Generator().manual_seed(15)
    for act in (None, "silu", "gelu"):
        def value(of):
            y = linear_act(of["x"], of["weight"], of["bias"], act, of["residual"])
            return (y.double() * gy.to(DEV)).sum(), (y * gy.to(DEV)).abs().sum().item()

        total, size = value(leaves)
        grads = dict(zip(leaves, torch.autograd.grad(total, list(leaves.values()))))
        for name in leaves:
            step = 2.0 ** -7
            way = torch.randn(t[name].shape, generator=gen).to(DEV)
            way = way / way.norm()
            with torch.no_grad():
                ends = [value(dict(leaves, **{name: leaves[name] + k * step * way}))[0].item() for k in (1, -1)]
            slope = (grads[name].double() * way).sum().item()
            assert abs((ends[0] - ends[1]) / (2 * step) - slope) <= 20 * step ** 2 + 4 * U * size / step, (act, name)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows", [7, 700])
def test_captured(rows, dtype):
    """Forward and backward captured, replayed with new inputs between eager ones."""
    from msda_opt2 import linear_act
    t, gy = _inputs(rows, 256, 512, TYPES[dtype], 16)
    still = {n: v.to(DEV).requires_grad_() for n, v in t.items()}
    g = gy.to(DEV)

    def step(of):
        y = linear_act(of["x"], of["weight"], of["bias"], "gelu", of["residual"])
        return [y.detach(), *torch.autograd.grad(y, list(of.values()), g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(still)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(still)
    for k in range(4):
        new, _ = _inputs(rows, 256, 512, TYPES[dtype], 20 + k)
        with torch.no_grad():
            for n, v in new.items():
                still[n].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step({n: v.to(DEV).requires_grad_() for n, v in new.items()})):
            assert torch.equal(a, b)


def test_two_streams():
    from msda_opt2 import linear_act
    t, _ = _inputs(4000, 256, 256, torch.bfloat16, 30)
    x, w = t["x"].to(DEV), t["weight"].to(DEV)
    want = linear_act(x, w)
    streams, out = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                out.append(linear_act(x, w))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in out)


def test_refusals_on_the_device():
    from msda_opt2 import linear_act
    x, w = torch.zeros(4, 8, device=DEV), torch.zeros(6, 8, device=DEV)
    for args, match in (((x, w.t()), "weight must be"), ((x, w.half()), "weight has dtype"), ((x, w.cpu()), "HIP"),
                        ((x, w, torch.zeros(8, device=DEV)), "bias must be"),
                        ((x, w, torch.zeros(6, device=DEV).half()), "bias has dtype"),
                        ((x, w, torch.zeros(6)), "HIP"), ((x, w, None, "tanh"), "act must be"),
                        ((x, w, None, None, x), "residual must be"),
                        ((x, w, None, None, torch.zeros(4, 6)), "HIP"),
                        ((x.double(), w.double()), "not implemented"), ((x[:, :0], w[:, :0]), "features"),
                        ((x, w[:0]), "features")):
        with pytest.raises(RuntimeError, match=match):
            linear_act(*args)
    x.requires_grad_()
    y = linear_act(x, w)
    g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
