"""The fp32 sums of group norm's backward and of the lookup's gradient against 64 bits, within the
bounds that the kernels' own order of additions gives (u = 2^-24 for each rounding; adding a first
term or a zero rounds nothing; e is the half step of the output's type).

Group norm, sums over positions: a thread adds up to 64 terms (63), eight lanes across leave three
steps between the lanes of a wave and three between the waves: 69 u of the sum of magnitudes, then
fp64. xh takes 5 u (x - mean in two floats, rstd, the product), its product with gz one more.

Lookup: up to 32 rows are added one after the other (k - 1). Of a row with more, a chunk's share is
at most 32 terms (31), and the chunks' sums come in runs by `groups` groups of lanes, which are then
added up. Scale and product: 2 u."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _near(got, ref, err, what):
    got = got.detach().cpu()
    half = torch.finfo(got.dtype).eps / 2
    bound = err + half * (ref.abs() + err) + torch.finfo(got.dtype).smallest_normal * half
    off = (got.double().reshape(ref.shape) - ref).abs()
    assert (off <= bound).all(), f"{what}: worst {(off / bound).max().item():.3f} of the bound"


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,positions,c,groups", [
    (512, 2048, 8, 2),   # 64 rounds of 32 positions of vectors
    (512, 256, 3, 1),    # 64 rounds of 4 positions of single channels
    (515, 2011, 8, 1), (2, 33, 64, 4)])
def test_group_norm_gradients(n, positions, c, groups, dtype):
    """512 images of one slab are as many tiles as are wanted: a tile is a whole image, 64 rounds
    of a thread. Gradients of one sign, so that no sum is small against its terms."""
    import modulated_deform_conv as mdc
    g = torch.Generator().manual_seed(n + c)
    x = (torch.randn(n, positions, c, generator=g) + 0.5).to(TYPES[dtype])
    gy = (0.5 + torch.rand(n, positions, c, generator=g)).to(TYPES[dtype])
    w, b = 1 + 0.3 * torch.randn(c, generator=g), torch.randn(c, generator=g)
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    y = mdc.group_norm_act_nhwc(leaves[0], groups, leaves[1], leaves[2])
    gx, gw, gb = torch.autograd.grad(y, leaves, gy.to(DEV))

    split = (n, positions, groups, c // groups)
    gz, d, wd = gy.double().view(split), x.double().view(split), w.double().view(split[2:])
    d = d - d.mean((1, 3), keepdim=True)
    r = 1 / torch.sqrt(d.square().mean((1, 3), keepdim=True) + 1e-5)
    xh, t = d * r, wd * gz
    p = gz * xh
    _near(gb, gz.sum((0, 1)), 69 * U * gz.abs().sum((0, 1)), "grad_bias")
    _near(gw, p.sum((0, 1)), 75 * U * p.abs().sum((0, 1)), "grad_weight")
    # by group: w, and the group's share and mean as fp32 values, one rounding each
    over = dict(dim=(1, 3), keepdim=True)
    m1, m2 = t.mean(**over), (t * xh).mean(**over)
    e1, e2 = 72 * U * t.abs().mean(**over), 78 * U * (t * xh).abs().mean(**over)
    # r (w gz - (m1 + xh m2)): each term's own roundings, and the three that follow
    err = r * (5 * U * t.abs() + e1 + 5 * U * m1.abs() + xh.abs() * e2 + 10 * U * (xh * m2).abs())
    _near(gx, r * (t - m1 - xh * m2), err, "grad_x")


def _additions(k, dim, dtype):
    """Roundings in the sums of rows with k places each."""
    size = torch.finfo(dtype).bits // 8
    vector = next((v // size for v in (16, 8) if dim * size % v == 0), 1)
    lanes = 1
    while lanes < 64 and lanes * vector < dim:
        lanes *= 2
    groups = 256 // lanes
    parts = k // 32 + 2  # chunks that a row touches, at most
    each = (parts + groups - 1) // groups
    many = 31 + (each - 1) + parts.clamp(max=groups) - 1
    return torch.where(k <= 32, (k - 1).clamp(min=0), many)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim", [1, 8, 33, 256, 1024])
def test_lookup_gradient(dim, dtype):
    """Rows of 0 to 96 places, of 100, 1,000 and 5,000, in a random order."""
    import _modulated_deform_conv_ext as ext
    g = torch.Generator().manual_seed(dim)
    k = torch.cat([torch.arange(97), torch.tensor([100, 1000, 5000, 0])])
    index = torch.arange(len(k)).repeat_interleave(k)
    index = index[torch.randperm(len(index), generator=g)]
    grad_out = (0.5 + torch.rand(len(index), dim, generator=g)).to(TYPES[dtype])
    grad = ext.embedding_backward(grad_out.to(DEV), index.to(DEV), len(k), 3.1)
    ref = 3.1 * torch.zeros(len(k), dim, dtype=torch.float64).index_add_(0, index, grad_out.double())
    _near(grad, ref, U * (_additions(k, dim, TYPES[dtype]) + 2).unsqueeze(1) * ref, "gradient")
