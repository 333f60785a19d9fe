"""What the training-side operators hand to the library, on the CPU: its entry points are replaced
by ones that record, so that nothing reaches a launch on any machine."""
import pytest
import torch

import _bevk
import _modulated_deform_conv_ext as ext
import modulated_deform_conv as mdc


@pytest.fixture
def recorded(monkeypatch):
    """The calls that reach the library, whatever device is current."""
    seen = []
    for name in ("bevk_clip_gradients", "bevk_embedding_forward", "bevk_group_norm_forward"):
        monkeypatch.setitem(_bevk._entries, name, lambda *a, name=name: seen.append(name) or 0)
    monkeypatch.setattr(_bevk, "_current_device", lambda: -1)
    monkeypatch.setattr(_bevk, "_raw_stream", lambda index: 0)
    return seen


def _cpu_layer():
    layer = torch.nn.Linear(4, 3)
    layer(torch.ones(2, 4)).sum().backward()
    return layer


@pytest.mark.parametrize("call", [
    lambda: mdc.clip_gradients_([torch.ones(3), torch.ones(2, 5)], 1.0),
    lambda: mdc.clip_gradients_(torch.ones(3), 1.0),
    lambda: mdc.clip_gradients_([torch.ones(3)], 1.0, out=[torch.zeros(3)]),
    lambda: mdc.clip_gradients_([torch.ones(3, 4).t()], 1.0),
    lambda: mdc.clip_gradients_([torch.ones(0)], 1.0),
    lambda: mdc.clip_grad_norm_(_cpu_layer().parameters(), 1.0),
    lambda: mdc.grad_norm([torch.ones(3), torch.ones(4)]),
    lambda: mdc.grad_norm(torch.ones(3, device="meta")),
    lambda: ext.clip_gradients([torch.ones(3)], 1.0)],
    ids=["list", "one", "out", "transposed", "empty", "layer", "norm", "meta", "ext"])
def test_gradients_off_the_gpu_are_refused(recorded, call):
    with pytest.raises(RuntimeError, match="expected tensors on a HIP"):
        call()
    assert not recorded


def test_a_gradient_off_the_gpu_among_others_is_refused(recorded):
    class OnDevice:
        is_cuda, layout, dtype, device = True, torch.strided, torch.float32, "cuda:0"
        shape, numel = torch.Size([3]), lambda self: 3
        get_device, data_ptr, is_contiguous = lambda self: 0, lambda self: 0x10000, lambda self: True

    for call in (lambda: ext.clip_gradients([OnDevice(), torch.ones(3)], 1.0),
                 lambda: ext.clip_gradients([torch.ones(3), OnDevice()], 1.0),
                 lambda: ext.clip_gradients([OnDevice()], 1.0, [torch.ones(3)])):
        with pytest.raises(RuntimeError, match="expected tensors on a HIP"):
            call()
    assert not recorded
