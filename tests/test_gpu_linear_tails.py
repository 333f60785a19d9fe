"""Activations far from zero, where they are small: right relative to their value. One feature of weight 1 without a
bias makes z the input itself.

Bounds, with u = 2^-24 and e the half step of the type: 16 bits: GELU's distribution below z 2.5e-5 of itself, its exponent
and that of SiLU rounded twice, (z^2 + 2 |z|) u, and 16 u for the rest; then e |y| and half of the least value of the type, or
of fp32 where that is larger (hardware exponentials and reciprocals keep no subnormals)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _exact(z, act):
    z = z.double()
    return z * (0.5 * torch.erfc(-z * 0.5 ** 0.5) if act == "gelu" else torch.sigmoid(z))  # (ndtr is 0 below -8.3)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows", [5, 400])
def test_16_bits(rows, dtype, act):
    """By the kernels for few rows and many."""
    from msda_opt2 import linear_act
    last = 14 if act == "gelu" else 86
    grid = torch.linspace(-last, last, 400 * 40, dtype=torch.float64).to(TYPES[dtype]).unique()
    w = torch.ones(1, 1, device=DEV, dtype=TYPES[dtype])
    z = grid.to(DEV)
    y = torch.cat([linear_act(part[:, None], w, None, act)[:, 0] for part in z.split(rows)]).double()
    want = _exact(z, act)
    rel = 2.5e-5 + (z.double() ** 2 + 2 * z.double().abs() + 16) * U
    e, least = torch.finfo(TYPES[dtype]).eps / 2, torch.finfo(TYPES[dtype]).smallest_normal
    bound = want.abs() * (rel + e + rel * e) + least * (e if dtype == "fp16" else 1) + z.double().abs() * 2.0 ** -126
    off = (y - want).abs()
    at = (off / bound).argmax()
    assert (off <= bound).all(), f"z {z[at].item()}: {y[at].item()} for {want[at].item()}"


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("rows", [5, 400, 4000])
def test_fp32(rows, act):
    from msda_opt2 import linear_act
    last = 12.9 if act == "gelu" else 86
    z = torch.linspace(-last, last, 40001, dtype=torch.float64).float().to(DEV).requires_grad_()
    w = torch.ones(1, 1, device=DEV)
    y = torch.cat([linear_act(part[:, None], w, None, act)[:, 0] for part in z.split(rows)])
    slope, = torch.autograd.grad(y.sum(), z)
    with torch.no_grad():
        d = z.double()
        if act == "gelu":
            terms = 0.5 * torch.erfc(-d * 0.5 ** 0.5), d * torch.exp(-0.5 * d * d) * (2 * torch.pi) ** -0.5
        else:
            terms = torch.sigmoid(d), d * torch.sigmoid(d) * torch.sigmoid(-d)
        least = (1 + d.abs()) * 2.0 ** -126
        for got, want, size, what in ((y, _exact(z, act), _exact(z, act).abs(), "y"),
                                      (slope, sum(terms), sum(t.abs() for t in terms), "slope")):
            off, bound = (got.double() - want).abs(), 16 * U * size + least
            at = (off / bound).argmax()
            assert (off <= bound).all(), f"{what} at z {d[at].item()}: {got[at].item()} for {want[at].item()}"
