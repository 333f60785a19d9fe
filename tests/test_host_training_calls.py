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


@pytest.fixture
def stand_ins(monkeypatch):
    """The library's calls behind the norm and the lookup, in plain torch."""
    monkeypatch.setattr(ext, "_group_norm_run", lambda x, *a: (x.clone(), None, None))
    monkeypatch.setattr(ext, "embedding_forward", lambda w, i, scale: w[i] * scale)


@pytest.mark.parametrize("grad", [True, False], ids=["grad", "no_grad"])
def test_forward_mode_is_refused(stand_ins, grad):
    """Neither operator has a forward-mode derivative: a tangent raises, with gradients recorded or
    not, and is never dropped. Without one both work within forward mode."""
    import msda_opt2
    import torch.autograd.forward_ad as fwd
    x, w, i = torch.randn(1, 2, 2, 4), torch.randn(4), torch.tensor([1, 0])
    table = torch.randn(3, 4)
    with torch.set_grad_enabled(grad), fwd.dual_level():
        def dual(t):
            return fwd.make_dual(t, torch.ones_like(t))

        for call in (lambda: mdc.group_norm_act_nhwc(dual(x), 2, w, w),
                     lambda: mdc.group_norm_act_nhwc(x, 2, dual(w), w),
                     lambda: mdc.group_norm_act_nhwc(x, 2, w, dual(w)),
                     lambda: mdc.GroupNormAct2d(2, 4)(dual(x.permute(0, 3, 1, 2))),
                     lambda: msda_opt2.embedding_lookup(dual(table), i)):
            with pytest.raises(NotImplementedError, match="jvp"):
                call()
        assert torch.equal(mdc.group_norm_act_nhwc(x, 2, w, w), x)
        assert torch.equal(msda_opt2.embedding_lookup(table, i, 2.0), 2 * table[i])


def test_calls_without_gradients_skip_the_bookkeeping(stand_ins, monkeypatch):
    import msda_opt2
    from modulated_deform_conv.group_norm import GroupNormActNHWCFunction
    for function in (GroupNormActNHWCFunction, msda_opt2.EmbeddingLookupFunction):
        monkeypatch.setattr(function, "forward", None)  # apply would fail
    with torch.no_grad():
        mdc.group_norm_act_nhwc(torch.ones(1, 2, 2, 4), 2)
        msda_opt2.embedding_lookup(torch.ones(3, 4), torch.tensor([1]))
