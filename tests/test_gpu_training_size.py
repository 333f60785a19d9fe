"""The training-side operators on tensors of more than 2^31 values (fp16, 4.3 GB each): offsets past
32 bits. Large inputs repeat a small one, so that the small one's results are the reference."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
TIMES, ROWS, C = 2050, 1024, 1024   # 2050 * 1024 * 1024 > 2^31
EPS = torch.finfo(torch.float16).eps


def _same(large, small, extra=0.0):
    """Every repetition within a step of fp16 of the small result (and extra)."""
    bound = EPS * small.float().abs() + extra + 2.0 ** -24
    for part in large.view(TIMES, ROWS, C).split(205):
        assert ((part.float() - small.view(1, ROWS, C).float()).abs() <= bound.view(1, ROWS, C)).all()


def test_group_norm():
    """Statistics, and so all values, are those of the small map; its parameters' gradients come
    TIMES as large. The fp32 means in grad_x differ by 64 * 2^-24 of terms whose mean magnitude is
    below 4 here."""
    import modulated_deform_conv as mdc
    torch.manual_seed(1)
    x, gy = (torch.randn(1, 32, 32, C, device=DEV).half() for _ in range(2))
    w, b = torch.randn(C, device=DEV).half(), torch.randn(C, device=DEV).half()

    def step(x, gy):
        leaves = [t.detach().requires_grad_() for t in (x, w.float(), b.float())]
        y = mdc.group_norm_act_nhwc(leaves[0], 32, leaves[1], leaves[2], 1e-5, "relu")
        return [y.detach(), *torch.autograd.grad(y, leaves, gy)]

    small = step(x, gy)
    large = step(x.view(1, ROWS, 1, C).repeat(1, TIMES, 1, 1), gy.view(1, ROWS, 1, C).repeat(1, TIMES, 1, 1))
    _same(large[0], small[0])
    _same(large[1], small[1], 8 * 64 * 2.0 ** -24 * 4)
    for a, s in zip(large[2:], small[2:]):
        assert ((a - TIMES * s).abs() <= 128 * 2.0 ** -24 * TIMES * ROWS * 4).all()


def test_embedding():
    import msda_opt2
    rows = TIMES * ROWS
    table = torch.zeros(rows, C, dtype=torch.float16, device=DEV)
    table[-3:] = torch.randn(3, C, device=DEV).half()
    index = torch.tensor([rows - 1, 5, rows - 3, -1, rows - 1, rows], device=DEV)
    leaf = table.requires_grad_()
    out = msda_opt2.embedding_lookup(leaf, index)
    assert torch.equal(out[0], table[-1]) and torch.equal(out[2], table[-3]) and torch.equal(out[4], table[-1])
    assert not out[[1, 3, 5]].any()
    g = torch.randn(6, C, device=DEV).half()
    grad, = torch.autograd.grad(out, leaf, g)
    assert torch.equal(grad[5], g[1]) and torch.equal(grad[-3], g[2]) and not grad[6:-3].any()
    assert torch.equal(grad[-1], (g[0].float() + g[4].float()).half()) and not grad[-2].any()
    many = torch.full((TIMES * ROWS,), -1, dtype=torch.int32, device=DEV)  # as many places, few rows
    many[-2:] = torch.tensor([2, 0], dtype=torch.int32)
    few = table[-3:].detach().clone().requires_grad_()
    out = msda_opt2.embedding_lookup(few, many)
    assert torch.equal(out[-2], few[2]) and torch.equal(out[-1], few[0]) and not out[-3].any()
    grad, = torch.autograd.grad(out, few, out)
    assert torch.equal(grad[[2, 0]], few[[2, 0]]) and not grad[1].any()


def test_clip():
    import modulated_deform_conv as mdc
    large = torch.full((TIMES * ROWS * C,), 0.5, dtype=torch.float16, device=DEV)
    other = torch.ones(1000, device=DEV)
    ref = (0.25 * large.numel() + 1000) ** 0.5
    norm = mdc.clip_gradients_([other, large], ref / 2)
    assert abs(norm.item() - ref) <= 2.0 ** -23 * ref
    assert (large.view(TIMES, -1) == 0.25).all() and ((other - 0.5).abs() <= 2.0 ** -23).all()
