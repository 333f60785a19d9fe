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
