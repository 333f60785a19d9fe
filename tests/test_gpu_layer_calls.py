"""Calls of the layer's operators that the documentation allows beside the usual ones: gradients in any order of strides,
forward mode (refused), a stream's gradient alone in another order."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _rand(g, *s):
    return torch.randn(*s, generator=g, device=DEV)


def test_linear_refuses_forward_mode():
    import torch.autograd.forward_ad as fwd

    from msda_opt2 import linear_act
    x, w = torch.randn(4, 32, device=DEV), torch.randn(8, 32, device=DEV)
    for at in (0, 1):
        with fwd.dual_level():
            args = [x, w]
            args[at] = fwd.make_dual(args[at], torch.ones_like(args[at]))
            with torch.no_grad(), pytest.raises(NotImplementedError):
                linear_act(*args)
            with pytest.raises(NotImplementedError):
                linear_act(*args, None, "gelu")


def _orders(t):
    """The same values: dense, transposed in memory, every second one of a larger tensor, off 16 bytes."""
    yield t.clone()
    yield t.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.empty(*t.shape[:-1], t.shape[-1] * 2, dtype=t.dtype, device=DEV)
    wide[..., ::2] = t
    yield wide[..., ::2]
    base = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
    base[1:] = t.flatten()
    yield base[1:].view(t.shape)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_norm_gradients_in_any_order(dtype):
    """Both gradients in each order against dense ones: the same values (off 16 bytes the sums have another order:
    a rounding of each)."""
    from msda_opt2 import residual_norm
    g = torch.Generator(device=DEV).manual_seed(4)
    x, r, gy, gs = (_rand(g, 6, 10, 64).to(dtype) for _ in range(4))
    leaves = [t.requires_grad_() for t in (x, r, _rand(g, 64), _rand(g, 64))]
    out = residual_norm(*leaves)
    want = torch.autograd.grad(out, leaves, (gy, gs), retain_graph=True)
    for a in _orders(gy):
        for b in _orders(gs):
            got = torch.autograd.grad(out, leaves, (a, b), retain_graph=True)
            for p, q in zip(got, want):
                if a.data_ptr() % 16 or b.data_ptr() % 16:
                    assert (p.float() - q.float()).abs().max() <= 2 * torch.finfo(dtype).eps * q.float().abs().max()
                else:
                    assert torch.equal(p, q)


@pytest.mark.parametrize("act", [None, "relu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_linear_gradients_in_any_order(dtype, act):
    from msda_opt2 import linear_act
    g = torch.Generator(device=DEV).manual_seed(5)
    leaves = [t.to(dtype).requires_grad_() for t in (_rand(g, 8, 9, 64), _rand(g, 72, 64) / 8, _rand(g, 72))]
    gy = _rand(g, 8, 9, 72).to(dtype)
    y = linear_act(*leaves, act)
    want = torch.autograd.grad(y, leaves, gy, retain_graph=True)
    for a in _orders(gy):
        for p, q in zip(torch.autograd.grad(y, leaves, a, retain_graph=True), want):
            if a.data_ptr() % 16:
                assert (p.float() - q.float()).abs().max() <= 2 * torch.finfo(dtype).eps * q.float().abs().max()
            else:
                assert torch.equal(p, q)
