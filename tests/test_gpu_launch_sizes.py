"""The training-side operators where one launch of a kernel would pass 2^32 work items: their
workgroups come in parts. Large inputs repeat a small one, whose 64-bit results and bounds are the
reference."""
import pytest
import torch

from test_gpu_group_norm import Reference, _half_step, _inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("times", [128, 257], ids=["one_part", "two_parts"])
def test_group_norm_of_many_images(times):
    """Single positions: 32 slabs an image, with 131,072 images 2^22 workgroups of 1,024 if it were
    one launch, and with 263,168 more than 2^23 tiles of 256 threads."""
    import modulated_deform_conv as mdc
    small = _inputs(1024, (1,), 1024, torch.float32, 31)
    r = Reference(*small, 32, "silu")
    x, gy = (t.to(DEV).repeat(times, 1, 1) for t in (small[0], small[3]))
    leaves = [x.requires_grad_(), *(t.to(DEV).requires_grad_() for t in small[1:3])]
    y = mdc.group_norm_act_nhwc(leaves[0], 32, leaves[1], leaves[2], 1e-5, "silu")
    grads = torch.autograd.grad(y, leaves, gy)
    half = _half_step(torch.float32)
    for got, ref, err in ((y.detach(), r.y, r.y_err), (grads[0], r.gx, r.gx_err)):
        ref, err = ref.to(DEV).view(1, 1024, 1024), err.to(DEV).view(1, 1024, 1024)
        bound = err + half * (ref.abs() + err) + torch.finfo(torch.float32).smallest_normal * half
        for part in got.view(times, 1024, 1024).split(32):
            assert ((part.double() - ref).abs() <= bound).all()
    for got, ref, err in ((grads[1], r.gw, r.gw_err), (grads[2], r.gb, r.gb_err)):
        ref, err = times * ref.flatten(), times * err.flatten()
        assert ((got.cpu().double() - ref).abs() <= err + half * (ref.abs() + err)).all()


def test_lookup_of_many_places():
    """1.07e10 single values: 10.5 million workgroups of 256 threads, in two parts."""
    import msda_opt2
    n = 2 ** 31 - 1024  # 7 * 306,783,232
    table = torch.randn(7, 5, device=DEV).half()
    index = torch.arange(n, dtype=torch.int32, device=DEV).remainder_(7)
    out = msda_opt2.embedding_lookup(table, index)
    assert out.shape == (n, 5)
    for part in out.view(-1, 7, 5).split(2 ** 24):
        assert (part == table).all()


def test_lookup_gradient_of_many_places():
    """268,436,000 places: more than 2^23 workgroups for chunks of 32. Small whole numbers, whose fp32
    sums (below 2^21) are exact."""
    import _modulated_deform_conv_ext as ext
    t = torch.arange(268_436_000, dtype=torch.int32, device=DEV)
    g = ((t % 1000) % 5 + (t // 1000) % 3).float().unsqueeze(1)
    grad = ext.embedding_backward(g, t.remainder_(1000), 1001)
    assert torch.equal(grad[:1000, 0].double(), g.view(-1, 1000).sum(0, dtype=torch.float64))
    assert not grad[1000:].any()


def test_lookup_gradient_of_a_large_table():
    """More than 2^30 rows: 2^22 workgroups of 1,024 for the sort, in two parts."""
    import _modulated_deform_conv_ext as ext
    rows = 2 ** 30 + 5
    index = torch.tensor([0, rows - 1, 5, -1, rows, 2 ** 30 - 1, rows - 1, 2 ** 22 - 1, 2 ** 21],
                         device=DEV)
    g = torch.arange(1, 10, device=DEV).half().unsqueeze(1)
    grad = ext.embedding_backward(g, index, rows)
    for row, value in ((0, 1), (rows - 1, 9), (5, 3), (2 ** 30 - 1, 6), (2 ** 22 - 1, 8), (2 ** 21, 9)):
        assert grad[row, 0].item() == value
        grad[row] = 0
    assert not grad.any()
