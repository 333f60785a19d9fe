"""The gradients of a projection in 16 bits have one rounding, however many rows there are: gz = gy act'(z) goes into
the products with 16 significant bits or more.

Bounds, with u = 2^-24 and e the half step of the type: the slope is off by its half step 2^-16, exp's and the formula's
roundings (below 32 u of 1.13) and what z's error does to it (its derivative is below 0.8; z's sum of K terms is (K / 4 +
28) u of their magnitudes off); gz then by 2^-16 of itself in bf16 (two values of 8 bits, each off by half a step: 2^-8 *
2^-8) and 2^-22 in fp16, or by half of fp16's least value; each product adds its terms' and its sum's errors, (terms / 16 +
64) u of the magnitudes; then e."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _inputs(rows, k, n, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rand(*s):
        return torch.randn(*s, generator=g, device=DEV)

    t = {"x": rand(rows, k).to(dtype), "weight": (rand(n, k) / k ** 0.5).to(dtype), "bias": rand(n).to(dtype)}
    return t, rand(rows, n).to(dtype)


def _gz(t, gy, act):
    """(gz, its error) in 64 bits."""
    d = {m: v.double() for m, v in t.items()}
    k = d["x"].shape[1]
    z = (d["x"] @ d["weight"].t() + d["bias"]).requires_grad_()
    gz, = torch.autograd.grad(getattr(torch.nn.functional, act)(z), z, gy.double())
    z_err = (k / 4 + 28) * U * (d["x"].abs() @ d["weight"].abs().t() + d["bias"].abs())
    two = torch.finfo(gy.dtype).eps ** 2 / 4 * gz.abs() + (2.0 ** -25 if gy.dtype == torch.float16 else 0)
    return gz, gy.double().abs() * (2.0 ** -16 + 32 * 1.13 * U + 0.8 * z_err) + two


def _inside(got, ref, err, what):
    e = torch.finfo(got.dtype).eps / 2
    bound = err + e * (ref.abs() + err) + torch.finfo(got.dtype).smallest_normal * e
    off = (got.double() - ref).abs()
    assert (off <= bound).all(), f"{what}: worst {(off / bound).max().item():.3f} of the bound"


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("size", [(17, 1, 1), (17, 64, 8), (33, 100, 75), (64, 256, 512), (65, 40, 129), (130, 64, 1024),
                                  (333, 72, 200), (500, 77, 1001), (640, 320, 256), (5001, 256, 128), (2000, 1024, 4096),
                                  (40000, 256, 512), (9001, 512, 264)], ids=str)
@pytest.mark.parametrize("dtype", list(TYPES))
def test_gradients_have_one_rounding(size, dtype, act):
    from msda_opt2 import linear_act
    rows, k, n = size
    t, gy = _inputs(rows, k, n, TYPES[dtype], sum(size))
    leaves = {m: v.clone().requires_grad_() for m, v in t.items()}
    gx, gw = torch.autograd.grad(linear_act(*leaves.values(), act), [leaves["x"], leaves["weight"]], gy)
    gz, gz_err = _gz(t, gy, act)
    x, w = t["x"].double(), t["weight"].double()
    for got, a, a_err, b, terms, what in ((gx, gz, gz_err, w, n, "x"), (gw, gz.t(), gz_err.t(), x, rows, "weight")):
        err = a_err @ b.abs()
        err = err + (terms / 16 + 64) * U * (a.abs() @ b.abs() + err)
        _inside(got, a @ b, err, f"gradient of {what}")


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_a_gz_past_the_type(act):
    """fp16: gy of the largest value where the slope is above 1: gz is past it, the gradients are not."""
    from msda_opt2 import linear_act
    rows, k, n, most = 40, 32, 64, 65504.0
    x = torch.full((rows, k), 1.5 / k, device=DEV).half()
    gy = torch.zeros(rows, n, device=DEV).half()
    gy[::2, 0] = most
    gy[::2, 1] = -most
    gy[1::2, 2] = -most
    gy[1::2, 3] = most / 2
    t = {"x": x, "weight": torch.full((n, k), 2.0 ** -6, device=DEV).half(),  # z 1.5: slopes of 1.04 and 1.13
         "bias": torch.full((n,), 1.5 - 1.5 / 64, device=DEV).half()}
    leaves = {m: v.clone().requires_grad_() for m, v in t.items()}
    gx, = torch.autograd.grad(linear_act(*leaves.values(), act), leaves["x"], gy)
    gz, gz_err = _gz(t, gy, act)
    assert gz.abs().max() > most
    b = t["weight"].double()
    err = gz_err @ b.abs()
    err = err + (n / 16 + 64) * U * (gz.abs() @ b.abs() + err)
    _inside(gx, gz @ b, err, "gradient of x")
