"""What a projection computes and keeps for its backward, by whose gradient is wanted: with stand-ins for the
kernels, on the CPU."""
import pytest
import torch

import msda_opt2.linear as mod


class _Ext:
    """Records whether the forward was asked for the slope."""

    def __init__(self):
        self.slopes, self.backwards = [], []

    def linear_forward(self, x, weight, bias=None, act=None, residual=None, with_slope=False):
        self.slopes.append(with_slope)
        y = x.detach() @ weight.detach().t()
        return y, torch.empty_like(y) if with_slope and act else None, (0,)

    def linear_backward(self, grad_y, x, weight, bias, slope, sizes, wanted):
        self.backwards.append(tuple(wanted))
        return (torch.zeros_like(x) if wanted[0] else None, torch.zeros_like(weight) if wanted[1] else None,
                torch.zeros_like(bias) if wanted[2] else None)


@pytest.fixture
def ext(monkeypatch):
    e = _Ext()
    monkeypatch.setattr(mod, "_loaded", e)
    return e


def _call(leaf=None):
    t = {"x": torch.zeros(4, 8), "weight": torch.zeros(6, 8), "bias": torch.zeros(6), "residual": torch.zeros(4, 6)}
    if leaf:
        t[leaf].requires_grad_()
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda v: kept.append(v) or v, lambda v: v):
        y = mod.linear_act(t["x"], t["weight"], t["bias"], "gelu", t["residual"])
    return t, y, kept


def test_nothing_to_differentiate(ext):
    """Grad mode is on, and no input records gradients."""
    _, y, kept = _call()
    assert ext.slopes == [False] and not kept and not y.requires_grad


def test_the_residual_alone(ext):
    t, y, kept = _call("residual")
    assert ext.slopes == [False] and not kept
    g = torch.randn(4, 6)
    assert torch.equal(torch.autograd.grad(y, t["residual"], g)[0], g) and not ext.backwards


@pytest.mark.parametrize("leaf,wanted", [("x", (True, False, False)), ("weight", (False, True, False)),
                                         ("bias", (False, False, True))])
def test_each_of_the_others(ext, leaf, wanted):
    t, y, kept = _call(leaf)
    assert ext.slopes == [True] and len(kept) == 4
    assert torch.autograd.grad(y, t[leaf], torch.ones(4, 6))[0].shape == t[leaf].shape
    assert ext.backwards == [wanted]
