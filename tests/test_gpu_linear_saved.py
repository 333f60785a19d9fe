"""What a projection keeps for its backward, seen by saved-tensor hooks: packing that is exact for numbers changes no
gradient, and values kept as whole numbers are in a tensor of whole numbers."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("act,residual", [(None, True), ("relu", False), ("relu", True), ("silu", True), ("gelu", False)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_floating_tensors_through_a_wider_type(dtype, act, residual, rows):
    """fp64 holds every number of the three types, and any NaN of one as some NaN."""
    from msda_opt2 import linear_act
    g = torch.Generator().manual_seed(rows)
    leaves = [torch.randn(*s, generator=g).to(TYPES[dtype]).to(DEV).requires_grad_() for s in ((rows, 64), (256, 64), (256,))]
    r = torch.randn(rows, 256, generator=g).to(TYPES[dtype]).to(DEV) if residual else None
    gy = torch.randn(rows, 256, generator=g).to(TYPES[dtype]).to(DEV)
    want = torch.autograd.grad(linear_act(*leaves, act, r), leaves, gy)

    def pack(t):
        return (t.double(), t.dtype) if t.is_floating_point() else (t.clone(), t.dtype)

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda kept: kept[0].to(kept[1])):
        y = linear_act(*leaves, act, r)
    got = torch.autograd.grad(y, leaves, gy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_saved_on_the_host():
    from msda_opt2 import linear_act
    g = torch.Generator().manual_seed(3)
    leaves = [torch.randn(*s, generator=g).bfloat16().to(DEV).requires_grad_() for s in ((100, 64), (256, 64), (256,))]
    gy = torch.randn(100, 256, generator=g).bfloat16().to(DEV)
    want = torch.autograd.grad(linear_act(*leaves, "gelu"), leaves, gy)
    with torch.autograd.graph.save_on_cpu():
        y = linear_act(*leaves, "gelu")
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, gy), want))
