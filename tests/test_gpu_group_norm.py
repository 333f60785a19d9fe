"""Group normalization with an activation (group_norm.hip) against the formulas in 64 bits.

Bounds, with u = 2^-24 and e the half step of the output type (finfo.eps / 2):
  z   x - mean, rstd, two products and a sum, each rounded once, on terms of |xh w| and |b|:
      6 u (|xh w| + |b|); the statistics are fp64
  y   ReLU adds nothing; SiLU has slope below 1.1 and is evaluated to 8 u: then e |y|
  gz  SiLU's derivative to 16 u (1 + |xh w| + |b|) of gy; ReLU's exactly (the sign of z is found
      in 64 bits)
  sums over positions: products to 3 u, fp32 sums of at most 48 terms in a row (serial and tree),
      then fp64: 64 u of the sum of magnitudes
  gx  three products of those, 6 u of each term, then e |gx|"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _inputs(n, hw, c, dtype, seed, ptype=None, mean=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, *hw, c, generator=g) * (0.3 + torch.rand(c, generator=g)) + mean
    w = 1 + 0.3 * torch.randn(c, generator=g)
    b = 0.3 * torch.randn(c, generator=g)
    gy = torch.randn(n, *hw, c, generator=g)
    return (x.to(dtype), w.to(ptype or dtype), b.to(ptype or dtype), gy.to(dtype))


class Reference:
    """The formulas in 64 bits, with the magnitudes that the bounds go by."""

    def __init__(self, x, w, b, gy, groups, act, eps=1e-5):
        n, c = x.shape[0], x.shape[-1]
        per = c // groups
        xd = x.double().reshape(n, -1, groups, per)
        w = (torch.ones(c) if w is None else w).double().view(groups, per)
        b = (torch.zeros(c) if b is None else b).double().view(groups, per)
        d = xd - xd.mean((1, 3), keepdim=True)
        r = 1 / torch.sqrt(d.square().mean((1, 3), keepdim=True) + eps)
        xh = d * r
        z = xh * w + b
        mag = (xh * w).abs() + b.abs()
        s = 1 / (1 + torch.exp(-z))
        if act == "relu":
            y, slope = torch.where(z <= 0, 0.0, z), torch.where(z <= 0, 0.0, 1.0)
        elif act == "silu":
            y, slope = z * s, s * (1 + z * (1 - s))
        else:
            y, slope = z, torch.ones_like(z)
        self.y, self.y_err = y, 6.6 * U * mag + 8 * U * y.abs()
        g = gy.double().reshape(z.shape)
        gz = g * slope
        gz_err = 16 * U * g.abs() * (1 + mag) if act == "silu" else torch.zeros_like(g)
        self.gw, self.gb = (gz * xh).sum((0, 1)), gz.sum((0, 1))
        self.gw_err = ((gz * xh).abs() * 64 * U + gz_err * xh.abs()).sum((0, 1))
        self.gb_err = (gz.abs() * 64 * U + gz_err).sum((0, 1))
        t, t_err = w * gz, w.abs() * gz_err
        m1, m2 = t.mean((1, 3), keepdim=True), (t * xh).mean((1, 3), keepdim=True)
        e1 = (64 * U * t.abs() + t_err).mean((1, 3), keepdim=True)
        e2 = ((64 * U * t.abs() + t_err) * xh.abs()).mean((1, 3), keepdim=True)
        self.gx = r * (t - m1 - xh * m2)
        self.gx_err = r * (t_err + e1 + xh.abs() * e2 + 6 * U * (t.abs() + m1.abs() + (xh * m2).abs()))
        self.shape = x.shape


def _near(got, ref, err, what):
    got = got.detach().cpu()
    tiny = torch.finfo(got.dtype).smallest_normal * _half_step(got.dtype)  # below, the step is fixed
    bound = err + (_half_step(got.dtype) * (ref.abs() + err)) + tiny
    off = (got.double().reshape(ref.shape) - ref).abs()
    assert (off <= bound).all(), f"{what}: worst {(off / bound).max().item():.3f} of the bound"


def _check(x, w, b, gy, groups, act, eps=1e-5):
    import modulated_deform_conv as mdc
    leaves = [t if t is None else t.to(DEV).requires_grad_() for t in (x, w, b)]
    y = mdc.group_norm_act_nhwc(leaves[0], groups, leaves[1], leaves[2], eps, act)
    assert y.shape == x.shape and y.dtype == x.dtype
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], gy.to(DEV))
    r = Reference(x, w, b, gy, groups, act, eps)
    _near(y, r.y, r.y_err, "y")
    _near(grads[0], r.gx, r.gx_err, "grad_x")
    rest = list(grads[1:])
    if w is not None:
        _near(rest.pop(0), r.gw, r.gw_err, "grad_weight")
    if b is not None:
        _near(rest.pop(0), r.gb, r.gb_err, "grad_bias")
    return y, grads


@pytest.mark.parametrize("act", [None, "relu", "silu"], ids=["none", "relu", "silu"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,hw,c,groups", [
    (1, (1, 1), 8, 2), (1, (1, 1), 3, 3), (2, (7, 9), 64, 8), (1, (15, 25), 256, 32),
    (3, (13, 17), 96, 32), (2, (11, 5), 75, 5), (1, (33, 31), 100, 25), (2, (9, 8), 256, 256),
    (2, (16, 16), 256, 1), (1, (29, 50), 512, 32), (6, (29, 50), 512, 32), (1, (70, 60), 40, 5),
    (5, (3, 1), 1000, 8), (2, (20, 21), 1040, 4), (1, (58, 100), 128, 32)])
def test_group_norm(n, hw, c, groups, dtype, act):
    _check(*_inputs(n, hw, c, TYPES[dtype], n * c + hw[0]), groups, act)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_fp32_parameters(dtype):
    x, w, b, gy = _inputs(2, (12, 10), 64, TYPES[dtype], 5, torch.float32)
    _, grads = _check(x, w, b, gy, 8, "relu")
    assert grads[1].dtype == torch.float32 and grads[2].dtype == torch.float32


@pytest.mark.parametrize("act", [None, "relu"])
@pytest.mark.parametrize("drop", [(1,), (2,), (1, 2)])
def test_without_parameters(drop, act):
    args = list(_inputs(2, (9, 7), 48, torch.float32, 6))
    for k in drop:
        args[k] = None
    _check(*args, 6, act)


def test_negative_and_zero_weights():
    x, w, b, gy = _inputs(2, (20, 20), 32, torch.float32, 7)
    w[::3] *= -1
    w[1::5] = 0
    _check(x, w, b, gy, 4, "relu")


def test_mean_far_from_zero():
    """A mean of 200 deviations costs no digits of y. The products' bound stays: x - mean is taken
    from the mean in two floats."""
    x, w, b, gy = _inputs(2, (31, 17), 64, torch.float32, 8, mean=130.0)
    _check(x, w, b, gy, 8, "silu")


def test_extreme_values():
    """Squares beyond fp32: 1e30 and 1e-30 as values (eps 0 for the small ones)."""
    x, w, b, gy = _inputs(1, (9, 9), 16, torch.float32, 9, mean=0.0)
    _check(x * 1e25, w, b, gy, 4, None)
    import modulated_deform_conv as mdc
    y = mdc.group_norm_act_nhwc((x * 1e-30).to(DEV), 4, w.to(DEV), b.to(DEV), 0.0, None)
    r = Reference(x * 1e-30, w, b, gy, 4, None, 0.0)
    _near(y, r.y, r.y_err, "y")


def test_constant_group():
    """Variance 0: y = act(b), and z = 0 has no gradient through ReLU."""
    import modulated_deform_conv as mdc
    x = torch.full((2, 5, 5, 16), 0.7, device=DEV, requires_grad=True)
    y = mdc.group_norm_act_nhwc(x, 4, None, None, 1e-5, "relu")
    gx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert not y.any() and not gx.any()


@pytest.mark.parametrize("act", [None, "relu", "silu"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_nonfinite_stays_in_its_group(bad, act):
    import modulated_deform_conv as mdc
    x, w, b, gy = _inputs(2, (40, 30), 64, torch.float32, 10)
    want, wg = _check(x, w, b, gy, 8, act)
    x[1, 3, 4, 17] = bad
    leaf = x.to(DEV).requires_grad_()
    y = mdc.group_norm_act_nhwc(leaf, 8, w.to(DEV), b.to(DEV), 1e-5, act)
    gx, = torch.autograd.grad(y, leaf, gy.to(DEV))
    for got, ref in ((y.detach(), want.detach()), (gx, wg[0])):
        assert got[1, ..., 16:24].isnan().all()
        got, ref = got.clone(), ref.clone()
        got[1, ..., 16:24] = ref[1, ..., 16:24] = 0
        assert torch.equal(got, ref)


def test_same_on_every_run():
    x, w, b, gy = _inputs(3, (58, 41), 256, torch.bfloat16, 11)
    a, ga = _check(x, w, b, gy, 32, "relu")
    c, gc = _check(x, w, b, gy, 32, "relu")
    assert torch.equal(a, c) and all(torch.equal(p, q) for p, q in zip(ga, gc))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_offset_views(dtype):
    """Inputs that start off a 16-byte boundary give what aligned ones give, within the bounds."""
    x, w, b, gy = _inputs(2, (10, 11), 64, TYPES[dtype], 12)
    import modulated_deform_conv as mdc

    def shifted(t):
        s = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape)
        return s.copy_(t).requires_grad_()

    leaves = [shifted(t) for t in (x, w, b)]
    y = mdc.group_norm_act_nhwc(leaves[0], 8, *leaves[1:], 1e-5, "silu")
    grads = torch.autograd.grad(y, leaves, shifted(gy).detach())
    r = Reference(x, w, b, gy, 8, "silu")
    for got, ref, err in zip((y, *grads), (r.y, r.gx, r.gw, r.gb),
                             (r.y_err, r.gx_err, r.gw_err, r.gb_err)):
        _near(got, ref, err, "offset view")


def test_other_strides_and_wanted_gradients():
    """A permuted input and an expanded gradient are made dense; only what is asked for comes."""
    import modulated_deform_conv as mdc
    x, w, b, _ = _inputs(2, (10, 11), 64, torch.float32, 13)
    xp = x.permute(0, 3, 1, 2).contiguous().to(DEV).permute(0, 2, 3, 1)
    assert not xp.is_contiguous()
    wl = w.to(DEV).requires_grad_()
    y = mdc.group_norm_act_nhwc(xp, 8, wl, b.to(DEV), 1e-5, "relu")
    y.backward(torch.ones(1, device=DEV).expand(y.shape))
    r = Reference(x, w, b, torch.ones(x.shape), 8, "relu")
    _near(y, r.y, r.y_err, "y")
    _near(wl.grad, r.gw, r.gw_err, "grad_weight")


@pytest.mark.parametrize("channels_last", [False, True])
def test_module(channels_last):
    import modulated_deform_conv as mdc
    x, w, b, gy = _inputs(2, (14, 9), 64, torch.float32, 14)
    m = mdc.GroupNormAct2d(8, 64, act="silu").to(DEV)
    with torch.no_grad():
        m.weight.copy_(w)
        m.bias.copy_(b)
    xn = x.permute(0, 3, 1, 2).to(DEV)
    xn = xn.contiguous(memory_format=torch.channels_last) if channels_last else xn.contiguous()
    xn.requires_grad_()
    y = m(xn)
    assert y.is_contiguous(memory_format=torch.channels_last if channels_last
                           else torch.contiguous_format)
    y.backward(gy.permute(0, 3, 1, 2).to(DEV))
    r = Reference(x, w, b, gy, 8, "silu")
    _near(y.permute(0, 2, 3, 1), r.y, r.y_err, "y")
    _near(xn.grad.permute(0, 2, 3, 1), r.gx, r.gx_err, "grad_x")
    _near(m.weight.grad, r.gw, r.gw_err, "grad_weight")


def test_empty():
    import modulated_deform_conv as mdc
    for shape in ((0, 4, 4, 16), (2, 0, 4, 16)):
        x = torch.empty(shape, device=DEV, requires_grad=True)
        w = torch.ones(16, device=DEV, requires_grad=True)
        y = mdc.group_norm_act_nhwc(x, 4, w, None, 1e-5, "relu")
        gx, gw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
        assert y.shape == gx.shape == x.shape and gw.shape == (16,) and not gw.any()


def test_differences():
    """The gradient against central differences of the 64-bit forward along random directions: the
    step's own error is step^2 |f'''|, below 1e-6 of the slope here."""
    x, w, b, gy = _inputs(1, (5, 6), 16, torch.float32, 15)
    _, grads = _check(x, w, b, gy, 4, "silu")
    g = torch.Generator().manual_seed(16)
    for k, t in enumerate((x, w, b)):
        v = torch.randn(t.shape, generator=g).double()

        def f(step):
            args = [x.double(), w.double(), b.double()]
            args[k] = args[k] + step * v
            r = Reference(*args, gy, 4, "silu")
            return (r.y * gy.double().reshape(r.y.shape)).sum().item()

        slope = (f(1e-4) - f(-1e-4)) / 2e-4
        terms = grads[k].detach().cpu().double() * v
        assert abs(terms.sum().item() - slope) <= 1e-5 * terms.abs().sum().item()


def test_graph_and_streams():
    """Captured training steps replayed on new inputs, with eager calls on another stream between
    the replays."""
    import modulated_deform_conv as mdc
    x, w, b, gy = (t.to(DEV) for t in _inputs(2, (30, 41), 64, torch.float16, 17))

    def step(x, w, b, gy):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = mdc.group_norm_act_nhwc(leaves[0], 8, leaves[1], leaves[2], 1e-5, "relu")
        return (y.detach(), *torch.autograd.grad(y, leaves, gy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, w, b, gy)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step(x, w, b, gy)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (18, 19, 20):
        new = [t.to(DEV) for t in _inputs(2, (30, 41), 64, torch.float16, seed)]
        for t, v in zip((x, w, b, gy), new):
            t.copy_(v)
        graph.replay()
        got = [o.clone() for o in outs]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = step(*new)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_deformable_layer_with_group_norm():
    """dcn_split_gn_nhwc is its two steps, with gradients for the parameters of both."""
    import modulated_deform_conv as mdc
    from modulated_deform_conv.dcn_split_nhwc import dcn_split_gn_nhwc, dcn_split_nhwc
    g = torch.Generator().manual_seed(21)

    def leaf(*size, s=1.0):
        return (s * torch.randn(*size, generator=g)).half().to(DEV).requires_grad_()

    x, w_off, b_off = leaf(2, 13, 15, 64), leaf(27, 64, 3, 3, s=0.02), leaf(27, s=0.3)
    w, gw, gb = leaf(64, 64, 3, 3, s=0.05), leaf(64), leaf(64, s=0.2)
    leaves = (x, w_off, b_off, w, gw, gb)
    out = dcn_split_gn_nhwc(x, w_off, b_off, w, None, 8, gw, gb)
    two = mdc.group_norm_act_nhwc(dcn_split_nhwc(x, w_off, b_off, w), 8, gw, gb, act="relu")
    gy = torch.randn(out.shape, generator=g).half().to(DEV)
    assert torch.equal(out, two)
    grads = torch.autograd.grad(out, leaves, gy)
    assert all(t.shape == v.shape and torch.isfinite(t).all() and t.any()
               for t, v in zip(grads, leaves))


def test_second_derivatives_are_refused():
    import modulated_deform_conv as mdc
    import msda_opt2
    x = torch.randn(1, 4, 4, 8, device=DEV, requires_grad=True)
    w = torch.randn(6, 8, device=DEV, requires_grad=True)
    i = torch.tensor([1, 2], device=DEV)
    for y, leaf in ((mdc.group_norm_act_nhwc(x, 2), x), (msda_opt2.embedding_lookup(w, i), w)):
        g, = torch.autograd.grad(y, leaf, torch.ones_like(y, requires_grad=True), create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


def test_many_tiles():
    """More slabs than tiles are wanted: shares of an image then go by the longest fp32 sum (64 of a
    thread), here with single channels, two to an image."""
    _check(*_inputs(31, (20, 15), 1041, torch.float16, 22), 3, "relu")
