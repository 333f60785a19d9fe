"""Calls of the layer's operators that the documentation allows beside the usual ones: gradients in any order of strides,
forward mode (refused), a stream's gradient alone in another order."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


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


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_norm_gradients_in_any_order(dtype):
    """Both gradients in each order of strides: the same bits as dense ones, and off 16 bytes (another order of sums)
    within the bounds of test_gpu_residual_norm.py."""
    import test_gpu_residual_norm as norm
    t, grads = norm._inputs((6, 10, 64), norm.TYPES[dtype], 4, "channels", True)
    leaves = {n: v.to(DEV).requires_grad_() for n, v in t.items()}
    from msda_opt2 import residual_norm
    out = residual_norm(leaves["x"], leaves["residual"], leaves["weight"], leaves["bias"], leaves["gate"], 0.5,
                        (leaves["block_weight"], leaves["block_bias"]))
    gy, gs = (g.to(DEV) for g in grads)
    want = torch.autograd.grad(out, list(leaves.values()), (gy, gs), retain_graph=True)
    r = norm.Reference(t, *grads, 0.5, True, "layer", 1e-5)
    for a in _orders(gy):
        for b in _orders(gs):
            got = torch.autograd.grad(out, list(leaves.values()), (a, b), retain_graph=True)
            for n, p, q in zip(leaves, got, want):
                if a.data_ptr() % 16 or b.data_ptr() % 16:
                    norm._near(p, *r.grads[n], n)
                else:
                    assert torch.equal(p, q), n


@pytest.mark.parametrize("act", [None, "relu", "gelu"])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_linear_gradients_in_any_order(dtype, act):
    """As above, with the bounds of test_gpu_linear.py."""
    import test_gpu_linear as lin
    from msda_opt2 import linear_act
    t, gy = lin._inputs(72, 64, 72, lin.TYPES[dtype], 5, False)
    leaves = [v.to(DEV).requires_grad_() for v in t.values() if v is not None]
    gy = gy.to(DEV)
    y = linear_act(*leaves, act)
    want = torch.autograd.grad(y, leaves, gy, retain_graph=True)
    r = lin.Reference(t, gy.cpu(), act)
    bounds = ((r.gx, r.gx_err), (r.gw, r.gw_err), (r.gb, r.gb_err))
    for a in _orders(gy):
        for p, q, bound in zip(torch.autograd.grad(y, leaves, a, retain_graph=True), want, bounds):
            if a.data_ptr() % 16:
                lin._near(p, *bound, "off 16 bytes")
            else:
                assert torch.equal(p, q)
