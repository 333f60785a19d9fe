"""AdamW where its second moment leaves fp32's normal numbers, and with a small or no eps, against 64 bits.

Bounds, with u = 2^-24: v is g^2 (1 - b2), of which a subnormal holds 2^-150 of half a step: v off by d = 2^-150 + 2^-150 / (1 -
b2) (1 - b2) (the square's own) + 4 u v, its root by d / (2 v) of itself and more where that is not small (sqrt(1 + x) - 1 is at
most x / 2 above and x below, for x in [-1, ...)); 10 u for the rest of the step, and p's own roundings 3 u |p|."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-19, 1e-8])
@pytest.mark.parametrize("g", [1e-22, 1e-21, 1e-20, 3e-20, 1e-19, 1e-18, 1e-15, 1e-4, 1e4, 1e18])
def test_first_step(g, eps):
    import modulated_deform_conv as mdc
    b1, b2, lr = 0.9, 0.999, 0.125
    p = torch.zeros(300, device=DEV)
    grad = torch.full((300,), g, device=DEV)
    grad[1::2] = -g
    state = mdc.adamw_state(p)
    mdc.adamw_step_(p, grad, state, lr=lr, betas=(b1, b2), eps=eps, weight_decay=0.0)
    d = grad.double()
    v = (1 - b2) * d * d
    up = lr * d / (torch.sqrt(v / (1 - b2)) + eps)
    off = (2.0 ** -150 * (1 + (1 - b2)) + 4 * U * v) / v  # of v
    rel = torch.where(off < 0.5, off, torch.inf) + 10 * U
    if eps > 0:  # where v is lost in its rounding, root is at most sqrt(2^-149 / (1 - b2)) and eps decides
        low = lr * d.abs() / ((torch.sqrt(v / (1 - b2)) + 2.0 ** -74 / (1 - b2) ** 0.5) + eps)
        high = lr * d.abs() / eps
        ok = ((p.double() + up).abs() <= rel * up.abs()) | ((p.abs() >= low * (1 - 10 * U)) & (p.abs() <= high * (1 + 10 * U)))
        assert ok.all()
        assert ((p <= 0) == (grad > 0)).all() or not p.any()
    elif off.max() < 0.5:
        assert ((p.double() + up).abs() <= rel * up.abs()).all(), (p[0].item(), up[0].item())
    elif (g * g) * (1 - b2) < 2.0 ** -150:  # v is 0: no step
        assert not p.any()


@pytest.mark.parametrize("eps", [0.0, 1e-45, 1e-39, 1e-38])
@pytest.mark.parametrize("bits", [32, 8])
def test_no_eps_and_no_gradient(bits, eps):
    """Moments of 0: a value decays and stays a number, also where eps is a subnormal."""
    import modulated_deform_conv as mdc
    p = torch.full((200,), 2.0, device=DEV)
    g = torch.zeros(200, device=DEV)
    g[7] = 0.5
    state = mdc.adamw_state(p, bits)
    for _ in range(2):
        mdc.adamw_step_(p, g, state, lr=0.125, eps=eps, weight_decay=0.5)
    want = torch.full((200,), 2.0 * (1 - 0.0625) ** 2, dtype=torch.float64, device=DEV)
    rest = torch.arange(200, device=DEV) != 7
    assert ((p.double() - want).abs() <= 4 * U * want)[rest].all()
    assert p.isfinite().all() and p[7] < want[7] - 0.2


def test_a_nan_moment_is_not_a_small_one():
    """v of NaN beside an m of a number: no step of m's size comes out of it."""
    import modulated_deform_conv as mdc
    p = torch.zeros(256, device=DEV)
    state = mdc.adamw_state(p)
    state["exp_avg"].fill_(0.5)
    state["exp_avg_sq"].fill_(1.0)
    state["exp_avg_sq"][5] = float("nan")
    mdc.adamw_step_(p, torch.full((256,), 0.5, device=DEV), state, lr=0.125, weight_decay=0.0)
    assert p[5].isnan() and p.isnan().sum() == 1
