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
