"""Projections, residual norms and the AdamW step on tensors of more than 2^31 values: offsets past 32 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ends(rows):
    """Some rows from all over, those around 2^31 values of 512 and the last ones."""
    return torch.cat([torch.arange(0, rows, rows // 50), torch.arange(2 ** 22 - 2, 2 ** 22 + 2),
                      torch.arange(rows - 40, rows)]).to(DEV)


@pytest.mark.parametrize("k", [64, 256])
def test_linear(k):
    """rows * N past 2^31; by tiles (K 64) and streamed rows (K 256); a bf16 sum of K products to
    (K / 16 + 28) u of its magnitudes, then half a step."""
    from msda_opt2 import linear_act
    rows, n = 2 ** 22 + 70_001, 512
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(rows, k, device=DEV, generator=gen, dtype=torch.bfloat16)
    w = (torch.randn(n, k, device=DEV, generator=gen) / k ** 0.5).bfloat16()
    b = torch.randn(n, device=DEV, generator=gen).bfloat16()
    y = linear_act(x, w, b, "relu", None)
    at = _ends(rows)
    z = x[at].double() @ w.double().t() + b.double()
    err = (k / 16 + 32) * 2.0 ** -24 * (x[at].double().abs() @ w.double().abs().t() + b.double().abs())
    got = y[at].double()
    assert ((got - z.clamp(min=0)).abs() <= err + 2.0 ** -8 * (z.abs() + err)).all()
    # gradients: rows that count are the last ones, so the weight's sum is theirs
    gy = torch.zeros_like(y)
    gy[-40:] = torch.randn(40, n, device=DEV, generator=gen).bfloat16()
    leaves = [t.requires_grad_() for t in (x, w, b)]
    gx, gw, gb = torch.autograd.grad(linear_act(*leaves, "relu"), leaves, gy)
    g = gy[-40:].double() * (y[-40:] > 0)
    for got, want, mag in ((gx[-40:], g @ w.double(), g.abs() @ w.double().abs()),
                           (gw, g.t() @ x[-40:].double(), g.abs().t() @ x[-40:].double().abs()),
                           (gb, g.sum(0), g.abs().sum(0))):
        e = (n / 16 + 64) * 2.0 ** -24 * mag
        assert ((got.double() - want).abs() <= e + 2.0 ** -8 * (want.abs() + e)).all()
    assert not gx[:-40].any()


def test_linear_fp32():
    from msda_opt2 import linear_act
    rows, k, n = 2 ** 22 + 70_001, 256, 512  # x of 4.4 GB, y of 8.7 GB
    gen = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(rows, k, device=DEV, generator=gen)
    w = torch.randn(n, k, device=DEV, generator=gen) / k ** 0.5
    at = _ends(rows)
    for weight in (w, w[:500]):  # streamed rows, and the tiled kernel for a part of the rows at a time
        y = linear_act(x, weight[:, :], None, None)
        z = x[at].double() @ weight.double().t()
        err = (k / 4 + 28) * 2.0 ** -24 * (x[at].double().abs() @ weight.double().abs().t())
        assert ((y[at].double() - z).abs() <= err).all()


def test_linear_fp32_large_weight():
    """A weight whose three bf16 pieces would pass 32-bit offsets."""
    from msda_opt2 import linear_act
    rows, k, n = 70, 2 ** 15, 2 ** 15 - 16
    gen = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn(rows, k, device=DEV, generator=gen).requires_grad_()
    w = (torch.randn(n, k, device=DEV, generator=gen) / k ** 0.5).requires_grad_()
    gy = torch.randn(rows, n, device=DEV, generator=gen)
    y = linear_act(x, w, None, "relu")
    gx, gw = torch.autograd.grad(y, [x, w], gy)
    with torch.no_grad():
        at = torch.cat([torch.arange(0, n, n // 60), torch.arange(n - 20, n)]).to(DEV)
        wd, xd = w[at].double(), x.double()
        z = xd @ wd.t()
        err = (k / 4 + 28) * 2.0 ** -24 * (xd.abs() @ wd.abs().t())
        assert ((y[:, at].double() - z.clamp(min=0)).abs() <= err).all()
        gz = gy.double() * (y > 0)
        back = torch.cat([torch.arange(0, k, k // 60), torch.arange(k - 20, k)]).to(DEV)
        wd = w[:, back].double()
        err = (n / 4 + 28) * 2.0 ** -24 * (gz.abs() @ wd.abs())
        assert ((gx[:, back].double() - gz @ wd).abs() <= err).all()
        err = (rows + 28) * 2.0 ** -24 * (gz[:, at].abs().t() @ xd.abs())
        assert ((gw[at].double() - gz[:, at].t() @ xd).abs() <= err).all()


def test_linear_weight_turned_in_parts():
    """A weight with more 64 x 64 pieces than one launch takes, turned for the gradient of x."""
    from msda_opt2 import linear_act
    rows, k, n = 5, 2 ** 15 + 2 ** 14, 2 ** 18  # 26 GB
    gen = torch.Generator(device=DEV).manual_seed(5)
    w = torch.empty(n, k, dtype=torch.bfloat16, device=DEV).normal_(generator=gen)
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    gy = torch.randn(rows, n, device=DEV, generator=gen).bfloat16()
    gx, = torch.autograd.grad(linear_act(x, w), x, gy)
    want = torch.zeros(rows, k, dtype=torch.float64, device=DEV)
    mag = want.clone()
    for a in range(0, n, 2 ** 14):
        part, g = w[a:a + 2 ** 14].double(), gy[:, a:a + 2 ** 14].double()
        want += g @ part
        mag += g.abs() @ part.abs_()
    err = (n / 16 + 64) * 2.0 ** -24 * mag
    assert ((gx.double() - want).abs() <= err + 2.0 ** -8 * (want.abs() + err)).all()


def test_linear_most_features():
    """As many features as there may be, of an odd number: gz, and its sums by columns, exact here."""
    from msda_opt2 import linear_act
    rows, k, n = 37, 16, 2 ** 24 - 1
    gen = torch.Generator(device=DEV).manual_seed(6)
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device=DEV)
    x[:, 0] = torch.randint(-4, 5, (rows,), device=DEV, generator=gen).bfloat16()
    w = torch.zeros(n, k, dtype=torch.bfloat16, device=DEV)
    w[:, 0] = torch.randint(-4, 5, (n,), device=DEV, generator=gen).bfloat16()
    b = torch.randint(-3, 4, (n,), device=DEV, generator=gen).float().requires_grad_()
    gy = torch.randint(-8, 9, (rows, n), device=DEV, generator=gen, dtype=torch.int8).bfloat16()
    y = linear_act(x, w, b, "relu")
    gb, = torch.autograd.grad(y, b, gy)
    for a in range(0, n, 2 ** 21):
        s = slice(a, a + 2 ** 21)
        z = x[:, :1].float() * w[s, 0].float() + b.detach()[s]
        assert torch.equal(y[:, s].float(), z.clamp(min=0))
        assert torch.equal(gb[s], (gy[:, s].float() * (z > 0)).sum(0))


def test_residual_norm():
    """Each repetition of a small input gives the small result; the parameters' gradients are TIMES as
    large, up to the fp32 sums' (TIMES * 1024 / 16 + 72) u of magnitudes below 4 in the mean."""
    from msda_opt2 import residual_norm
    times, rows, c = 2050, 1024, 1024
    gen = torch.Generator(device=DEV).manual_seed(3)
    small = [torch.randn(1, rows, c, device=DEV, generator=gen).half() for _ in range(4)]
    params = [torch.randn(c, device=DEV, generator=gen) for _ in range(3)]

    def step(x, r, gy, gs):
        leaves = [t.detach().requires_grad_() for t in (x, r, *params)]
        out = residual_norm(leaves[0], leaves[1], leaves[2], leaves[3], gate=leaves[4], scale=0.5)
        return [*(o.detach() for o in out), *torch.autograd.grad(out, leaves, (gy, gs))]

    want = step(*small)
    got = step(*(t.repeat(1, times, 1) for t in small))
    for a, s in zip(got[:4], want[:4]):
        for part in a.view(times, rows, c).split(205):
            assert torch.equal(part, s.view(1, rows, c).expand_as(part))
    for a, s in zip(got[4:], want[4:]):
        assert ((a - times * s).abs() <= (times * rows / 16 + 72) * 2.0 ** -24 * times * rows * 4).all()
        assert ((a / times - s).norm() / s.norm()).item() <= 1e-3


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw(bits):
    """One tensor past 2^31 values and a small one behind it: what the first step gives everywhere."""
    import modulated_deform_conv as mdc
    n = 2 ** 31 + 1001
    p = [torch.ones(n, device=DEV), torch.ones(7, device=DEV)]
    g = [torch.empty(n, dtype=torch.bfloat16, device=DEV).fill_(0.25), torch.full((7,), -0.5, device=DEV)]
    g[0][1::2] = -2.0
    state = mdc.adamw_state(p, bits)
    mdc.adamw_step_(p, g, state, lr=0.125, weight_decay=0.0)
    # m / sqrt(v) is the gradient's sign after one step, to the roundings of both and of the factors
    for part, k in ((p[0][:2 ** 20], 0), (p[0][2 ** 31 - 2 ** 19:], 0)):
        want = torch.where(g[0][:2].float() > 0, 1 - 0.125, 1 + 0.125)
        assert ((part[:part.numel() // 2 * 2].view(-1, 2) - want).abs() <= 0.125 * 16 * 2.0 ** -24 + 2.0 ** -23).all()
    assert ((p[1] - 1.125).abs() <= 0.125 * 16 * 2.0 ** -24 + 2.0 ** -23).all()
    assert state["exp_avg"].numel() == (n + 127) // 128 * 128 + 128
    if bits == 32:
        assert torch.equal(state["exp_avg"][n - 1001:n - 1], state["exp_avg"][:1000])
        assert not state["exp_avg"][n:n + 23].any()
    else:  # rounded at random: every value is one of the two codes around it, and the scale is the largest's
        from itertools import islice
        scale = state["exp_avg_scale"]
        assert (scale[:-2] == scale[0]).all() and set(islice(state["exp_avg"][2 ** 31:2 ** 31 + 500].tolist(), 500)) \
            <= set(state["exp_avg"][:2 ** 16].tolist())
        v = mdc.adamw_moments({k: (t[-2 ** 12:] if k.startswith("exp_avg") and "scale" not in k else
                                   t[-2 ** 5:] if "scale" in k else t) for k, t in state.items()})[1]
        assert v[-128:-121].min() > 0 and not v[-121:].any()
