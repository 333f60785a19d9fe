"""Refusals of the AdamW step on the CPU, in Python and at the C ABI: nothing here reaches a launch
(fake device addresses are never followed)."""
import ctypes

import pytest
import torch

import _bevk
import modulated_deform_conv as mdc

INVALID, UNSUPPORTED = 1, 2
P = 0x10000


def _err():
    return _bevk.lib().bevk_last_error().decode()


def test_needs_a_device():
    p, g = [torch.zeros(4)], [torch.zeros(4)]
    state = mdc.adamw_state(p)
    with pytest.raises(RuntimeError, match="HIP"):
        mdc.adamw_step_(p, g, state, lr=0.1)
    with pytest.raises(RuntimeError, match="no parameters"):
        mdc.adamw_step_([], [], state, lr=0.1)
    with pytest.raises(RuntimeError, match="2 gradients for 1"):
        mdc.adamw_step_(p, g * 2, state, lr=0.1)
    with pytest.raises(RuntimeError, match="parameter 0 has no gradient"):
        mdc.adamw_step_(p, [None], state, lr=0.1, max_norm=1.0)
    with pytest.raises(RuntimeError, match="8 or 32"):
        mdc.adamw_state(p, bits=16)
    with pytest.raises(RuntimeError, match="no parameters"):
        mdc.adamw_state([])
    with pytest.raises(RuntimeError, match="seed"):
        mdc.adamw_state(p, seed=-1)


def _on_device(step):
    """The parts of a call that are checked before the device's own."""
    class Fake:
        def __init__(self, t): self.t = t
        def __getattr__(self, n): return getattr(self.t, n)
        def get_device(self): return 0
        is_cuda = True
    return Fake(step)


@pytest.mark.parametrize("seed", [-1, 2 ** 64, 1.0, "1"])
def test_refuses_a_loaded_seed(seed, monkeypatch):
    import _modulated_deform_conv_ext as ext
    monkeypatch.setattr(ext, "_grad_arrays", lambda fn, tensors, device: (None, None, True))
    p = _on_device(torch.zeros(4))
    with pytest.raises(RuntimeError, match="seed"):
        ext.adamw_step([p], [p], {"seed": seed}, 0.1, 0.9, 0.99, 1e-8, 0.0)


def test_state_layout():
    p = [torch.zeros(4), torch.zeros(128), torch.zeros(0), torch.zeros(3, 50)]
    state = mdc.adamw_state(p, 8, seed=7)
    assert state["exp_avg"].shape == state["exp_avg_sq"].shape == (128 + 128 + 256,)
    assert state["exp_avg_scale"].shape == (4,) and state["step"].tolist() == [0] and state["seed"] == 7
    assert mdc.adamw_state(p)["exp_avg"].dtype == torch.float32


def _step(count=1, ps=(P,), pt=(0,), gs=(0x20000,), gt=(0,), cs=None, ct=None, ns=(128,), bits=32, m=0x30000,
          v=0x40000, ms=0x50000, vs=0x60000, values=128, step=0x70000, lr=0.1, b1=0.9, b2=0.999, eps=1e-8,
          wd=0.0, norm=None, max_norm=0.0, ws=0x80000, wb=64):
    def arr(t, a):
        return None if a is None else (t * len(a))(*a)
    u64, i32, i64 = ctypes.c_uint64, ctypes.c_int, ctypes.c_int64
    return _bevk.lib().bevk_adamw_step(
        count, arr(u64, ps), arr(i32, pt), arr(u64, gs), arr(i32, gt), arr(u64, cs), arr(i32, ct), arr(i64, ns),
        bits, m, v, ms, vs, values, step, 0, lr, None, b1, b2, eps, wd, norm, max_norm, ws, wb, None)


@pytest.mark.parametrize("kw,code,match", [
    (dict(count=-1), INVALID, "negative count"), (dict(ns=(-1,)), INVALID, "negative size"),
    (dict(ns=(2 ** 41,)), INVALID, "2\\^40"), (dict(bits=16), INVALID, "8 or 32"),
    (dict(pt=(3,)), UNSUPPORTED, "Double"), (dict(gt=(3,)), UNSUPPORTED, "Double"),
    (dict(cs=(0x90000,), ct=(7,)), UNSUPPORTED, "unknown"), (dict(ps=None), INVALID, "null array"),
    (dict(cs=(0x90000,)), INVALID, "null array"), (dict(ps=(0,)), INVALID, "null tensor"),
    (dict(gs=(0,)), INVALID, "null tensor"), (dict(step=None), INVALID, "null tensor"),
    (dict(m=None), INVALID, "null tensor"), (dict(bits=8, ms=None), INVALID, "null tensor"),
    (dict(ps=(P + 2,)), INVALID, "aligned to its type"), (dict(m=0x30008), INVALID, "16-byte"),
    (dict(values=256), INVALID, "need 128"), (dict(values=0), INVALID, "need 128"),
    (dict(lr=-1.0), INVALID, "negative"), (dict(lr=float("nan")), INVALID, "negative"),
    (dict(b1=1.0), INVALID, "betas"), (dict(b2=-0.1), INVALID, "betas"), (dict(wd=-1.0), INVALID, "negative"),
    (dict(max_norm=1.0), INVALID, "null tensor"), (dict(norm=0xA0000, max_norm=-1.0), INVALID, "negative"),
    (dict(wb=8), INVALID, "workspace too small"), (dict(ws=None), INVALID, "null tensor"),
    (dict(ws=0x80008), INVALID, "16-byte"),
    (dict(gs=(P,)), INVALID, "overlaps"), (dict(gs=(P + 508,)), INVALID, "overlaps"),
    (dict(m=P), INVALID, "overlap"), (dict(m=0x30000, v=0x30100), INVALID, "overlap"),
    (dict(cs=(P + 256,), ct=(2,)), INVALID, "overlap"), (dict(step=P + 8), INVALID, "overlap"),
    (dict(norm=0x30004, max_norm=1.0), INVALID, "overlaps"), (dict(ws=P), INVALID, "overlap"),
    (dict(count=2, ps=(P, P + 508), pt=(0, 0), gs=(0x20000, 0x28000), gt=(0, 0), ns=(128, 5), values=256),
     INVALID, "overlap")])
def test_refusals(kw, code, match):
    import re
    assert _step(**kw) == code and re.search(match, _err()), _err()


def test_moments_refusals():
    f = _bevk.lib().bevk_adamw_moments
    assert f(P, P, 0, 128, 1, P, None) == UNSUPPORTED
    assert f(P, P, 0, 100, 0, P, None) == INVALID and "multiple" in _err()
    assert f(P, P, 0, -128, 0, P, None) == INVALID
    assert f(None, P, 0, 128, 0, P, None) == INVALID and "null" in _err()
    assert f(P + 8, P, 0, 128, 0, P, None) == INVALID and "16-byte" in _err()
    assert f(None, None, 0, 0, 0, None, None) == 0
