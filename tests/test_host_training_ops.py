"""Refusals of the training-side operators on the CPU, in Python and at the C ABI: nothing here
reaches a launch (fake device addresses are never followed)."""
import ctypes

import pytest
import torch

import _bevk
import _modulated_deform_conv_ext as ext
import modulated_deform_conv as mdc

INVALID, UNSUPPORTED = 1, 2
P = ctypes.c_void_p(0x10000)


def _err():
    return _bevk.lib().bevk_last_error().decode()


def _meta(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="meta")


@pytest.fixture
def no_device_check(monkeypatch):
    monkeypatch.setattr(_bevk, "require_device", lambda fn, *t: 0)


def test_group_norm_needs_a_device():
    with pytest.raises(RuntimeError, match="HIP"):
        mdc.group_norm_act_nhwc(torch.zeros(1, 4, 4, 8), 2)
    with pytest.raises(ValueError, match="4D"):
        mdc.GroupNormAct2d(2, 8)(torch.zeros(1, 4, 8))
    with pytest.raises(ValueError, match="divisible"):
        mdc.GroupNormAct2d(3, 8)
    with pytest.raises(ValueError, match="act"):
        mdc.GroupNormAct2d(2, 8, act="tanh")


def test_group_norm_refusals(no_device_check):
    x = _meta(2, 4, 4, 8)
    f = ext.group_norm_forward
    for bad, match in (((_meta(2, 8), 2, None, None), "positions"),
                       ((x.permute(0, 3, 1, 2), 2, None, None), "contiguous"),
                       ((x, 3, None, None), "divisible"), ((x, 0, None, None), "divisible"),
                       ((x, 2, _meta(4), None), r"weight must be \[8\]"),
                       ((x, 2, None, _meta(8, dtype=torch.float16)), "bias has dtype"),
                       ((x.half(), 2, _meta(8), _meta(8, dtype=torch.float16)), "one dtype"),
                       ((x.double(), 2, None, None), "not implemented"),
                       ((_meta(1, 1, 2 ** 31), 2, None, None), "2\\^30 channels"),
                       ((x.long(), 2, None, None), "not supported")):
        with pytest.raises(RuntimeError, match=match):
            f(*bad, 1e-5, None)
    with pytest.raises(RuntimeError, match="act must be"):
        f(x, 2, None, None, 1e-5, "gelu")
    b = ext.group_norm_backward
    stats = _meta(2, 2, 2, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="grad_y"):
        b(_meta(2, 4, 4, 4), x, 2, None, None, None, stats)
    with pytest.raises(RuntimeError, match="grad_y has dtype"):
        b(x.half(), x, 2, None, None, None, stats)
    with pytest.raises(RuntimeError, match="stats"):
        b(x, x, 2, None, None, None, _meta(2, 2, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="stats must be float64"):
        b(x, x, 2, None, None, None, _meta(2, 2, 2))


def test_group_norm_c_abi():
    lib = _bevk.lib()

    def fwd(dtype=0, x=P, w=None, b=None, pd=0, n=1, p=4, c=8, g=2, eps=1e-5, act=0, ws=P, wb=1 << 30,
            y=P, st=P):
        return lib.bevk_group_norm_forward(dtype, x, w, b, pd, n, p, c, g, eps, act, ws, wb, y, st, None)

    assert fwd(dtype=3) == UNSUPPORTED and "Double" in _err()
    assert fwd(dtype=9) == UNSUPPORTED
    assert fwd(dtype=1, pd=2) == INVALID and "type" in _err()
    assert fwd(c=9) == INVALID and "divisible" in _err()
    for kw in (dict(n=0), dict(p=0), dict(c=0), dict(g=0), dict(n=-1)):
        assert fwd(**kw) == INVALID and "positive" in _err()
    assert fwd(n=1 << 30, p=1 << 30) == INVALID and "2^40" in _err()
    assert fwd(c=(1 << 30) + 2) == INVALID and "2^30" in _err()
    assert fwd(act=3) == INVALID and "activation" in _err()
    assert fwd(eps=-1.0) == INVALID and "eps" in _err()
    assert fwd(eps=float("nan")) == INVALID and "eps" in _err()
    for kw in (dict(x=None), dict(y=None)):
        assert fwd(**kw) == INVALID and "null" in _err()

    def bwd(dtype=0, gy=P, x=P, act=0, st=P, ws=P, wb=1 << 30, gx=P):
        return lib.bevk_group_norm_backward(dtype, gy, x, None, None, dtype, 2, 4, 8, 2, act, st, ws, wb,
                                            gx, None, None, None)

    assert bwd(dtype=3) == UNSUPPORTED
    for kw in (dict(gy=None), dict(x=None), dict(st=None), dict(ws=None)):
        assert bwd(**kw) == INVALID and "null" in _err()
    assert bwd(wb=0) == INVALID and "workspace" in _err()
    assert bwd(ws=ctypes.c_void_p(0x10008)) == INVALID and "16-byte" in _err()
    assert bwd(gx=None) == 0                            # nothing wanted
    ws = lib.bevk_group_norm_workspace_bytes
    assert ws(3, 0, 1, 4, 8, 2, 1) == -1 and ws(0, 0, 1, 4, 9, 2, 1) == -1
    assert ws(0, 1, 1, 4, 8, 2, 1) > 0 and ws(0, 0, 1, 4000, 8, 2, 1) > 0
    assert ws(0, 0, 1, 4, 8, 2, 1) == 0                # one launch without a workspace


def test_embedding_refusals(no_device_check):
    import msda_opt2
    w, i = _meta(10, 8), _meta(3, 4, dtype=torch.int64)
    for bad, match in (((_meta(10), i), r"weight must be \[V, D\]"), ((w, i.float()), "int64 or int32"),
                       ((w, i.short()), "int64 or int32"), ((w.t(), i), "contiguous"),
                       ((w, i.t()), "contiguous"), ((w.long(), i), "not supported"),
                       ((w.double(), i), "not implemented"),
                       ((_meta(1, 2 ** 32 + 8), i), "2\\^30 channels")):
        with pytest.raises(RuntimeError, match=match):
            ext.embedding_forward(*bad)
    g = _meta(3, 4, 8)
    for bad, match in (((g, _meta(12, dtype=torch.int64), 10), "grad_out must be"),
                       ((_meta(3, 8), i, 10), "grad_out must be"),
                       ((g, i, 10, 1.0, 10), "padding_idx"), ((g, i, 10, 1.0, -1), "padding_idx"),
                       ((g.double(), i, 10), "not implemented"), ((g, i, -1), "not implemented")):
        with pytest.raises(RuntimeError, match=match):
            ext.embedding_backward(*bad)
    for padding in (-1, 10):
        with pytest.raises(RuntimeError, match="padding_idx"):
            msda_opt2.embedding_lookup(w, i, 1.0, padding)


def test_embedding_needs_a_device():
    import msda_opt2
    with pytest.raises(RuntimeError, match="HIP"):
        msda_opt2.embedding_lookup(torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64))


def test_embedding_c_abi():
    lib = _bevk.lib()

    def fwd(dtype=0, w=P, rows=10, dim=8, i=P, n=4, out=P):
        return lib.bevk_embedding_forward(dtype, w, rows, dim, i, 1, n, 1.0, out, None)

    assert fwd(dtype=3) == UNSUPPORTED and "Double" in _err()
    for kw in (dict(n=-1), dict(rows=-1), dict(dim=-1)):
        assert fwd(**kw) == INVALID and "negative" in _err()
    for kw in (dict(n=1 << 31), dict(rows=1 << 31)):
        assert fwd(**kw) == INVALID and "2^31" in _err()
    for kw in (dict(w=None), dict(i=None), dict(out=None)):
        assert fwd(**kw) == INVALID and "null" in _err()
    assert fwd(n=0) == 0 and fwd(dim=0) == 0

    def bwd(dtype=0, g=P, i=P, n=4, rows=10, dim=8, padding=-1, ws=P, wb=1 << 30, gw=P):
        return lib.bevk_embedding_backward(dtype, g, i, 1, n, rows, dim, 1.0, padding, ws, wb, gw, None)

    assert bwd(dtype=9) == UNSUPPORTED
    for padding in (-2, 10):
        assert bwd(padding=padding) == INVALID and "padding_idx" in _err()
    for kw in (dict(g=None), dict(i=None), dict(gw=None)):
        assert bwd(**kw) == INVALID and "null" in _err()
    assert bwd(wb=0) == INVALID and "workspace" in _err()
    assert bwd(ws=ctypes.c_void_p(0x10004)) == INVALID and "16-byte" in _err()
    assert bwd(dim=(1 << 30) + 1) == INVALID and "2^30" in _err()
    assert bwd(rows=0) == 0 and bwd(dim=0) == 0
    ws = lib.bevk_embedding_backward_workspace_bytes
    assert ws(3, 4, 10, 8) == -1 and ws(0, -1, 10, 8) == -1 and ws(0, 1 << 31, 10, 8) == -1


def test_clip_refusals(monkeypatch):
    f = ext.clip_gradients
    with pytest.raises(RuntimeError, match="HIP"):
        mdc.clip_gradients_([torch.zeros(3)], 1.0)
    with pytest.raises(RuntimeError, match="HIP"):
        mdc.grad_norm(torch.zeros(3))
    for bad in (-1.0, float("nan")):
        with pytest.raises(RuntimeError, match="max_norm"):
            mdc.clip_gradients_([torch.zeros(3)], bad)
    with pytest.raises(RuntimeError, match="outputs for 0"):
        mdc.clip_gradients_([], 1.0, out=[torch.zeros(3)])

    class Fake:  # a device tensor's attributes without a device
        is_cuda, layout, device = True, torch.strided, "cuda:0"

        def __init__(self, t, index=0):
            self.t, self.index = t, index
            self.dtype, self.shape = t.dtype, t.shape

        def get_device(self):
            return self.index

        def data_ptr(self):
            return 0x10000

        def __getattr__(self, name):
            return getattr(self.t, name)

    a = Fake(torch.zeros(4, 6))
    for bad, match in (([a, Fake(torch.zeros(2), 1)], "different devices"),
                       ([Fake(torch.zeros(4, 6)[:, :3])], "dense"),
                       ([Fake(torch.zeros(4, 1).expand(4, 6))], "dense"),
                       ([Fake(torch.zeros(4).long())], "not supported")):
        with pytest.raises(RuntimeError, match=match):
            f(bad, 1.0)
    for out, match in (([], "0 outputs for 1"), ([Fake(torch.zeros(6, 4))], "an output has shape"),
                       ([Fake(torch.zeros(6, 4).t())], "an output has shape")):
        with pytest.raises(RuntimeError, match=match):
            f([a], 1.0, out)


def test_clip_c_abi():
    lib = _bevk.lib()

    def call(types=(0, 1), sizes=(100, 50), at=(0x10000, 0x20000), out=None, out_types=None, max_norm=1.0,
             ws=P, wb=1 << 30, norm=P):
        n = len(sizes)
        arr = lambda t, v: None if v is None else (t * n)(*v)  # noqa: E731
        return lib.bevk_clip_gradients(n, arr(ctypes.c_void_p, at), arr(ctypes.c_int, types),
                                       arr(ctypes.c_int64, sizes), arr(ctypes.c_void_p, out),
                                       arr(ctypes.c_int, out_types), max_norm, ws, wb, norm, None)

    assert call(types=(0, 3)) == UNSUPPORTED and "Double" in _err()
    assert call(sizes=(-1, 5)) == INVALID and "negative" in _err()
    assert call(sizes=(1 << 40, 1)) == INVALID and "2^40" in _err()
    assert call(at=(0x10000, 0)) == INVALID and "null" in _err()
    assert call(at=(0x10002, 0x20000)) == INVALID and "aligned" in _err()
    assert call(norm=None) == INVALID and "null" in _err()
    assert call(at=None) == INVALID and "null" in _err()
    assert call(ws=None) == INVALID and "null" in _err()
    assert call(wb=8) == INVALID and "workspace" in _err()
    both = dict(out=(0x10000, 0x20000), out_types=(0, 1))
    for bad in (-1.0, float("nan")):
        assert call(**both, max_norm=bad) == INVALID and "max_norm" in _err()
    assert call(out=(0x30000, 0x30000 + 396), out_types=(0, 1)) == INVALID and "two outputs" in _err()
    assert call(out=(0x10000, 0x10100), out_types=(0, 1)) == INVALID and "overlap" in _err()
    assert call(out=(0x10004, 0x20000), out_types=(0, 1)) == INVALID and "not its own" in _err()
    assert call(out=(0x20000, 0x10000), out_types=(0, 1)) == INVALID and "not its own" in _err()
    assert call(out=(0x10000, 0x20000), out_types=(0, 0)) == INVALID and "not its own" in _err()
    assert lib.bevk_clip_gradients(-1, None, None, None, None, None, 1.0, P, 8, P, None) == INVALID
    ws = lib.bevk_clip_gradients_workspace_bytes
    assert ws(0, None) == 0 and ws(-1, None) == -1 and ws(1, None) == -1
    assert ws(2, (ctypes.c_int64 * 2)(1, 0)) == 8


def test_calls_go_to_the_tensors_device(monkeypatch):
    """A call for tensors of another device than the current one makes theirs current for the call,
    and passes that device's stream."""
    import contextlib
    current, seen = [0], []

    @contextlib.contextmanager
    def device(index):
        before, current[0] = current[0], index
        yield
        current[0] = before

    monkeypatch.setattr(_bevk, "_current_device", lambda: current[0])
    monkeypatch.setattr(_bevk, "_raw_stream", lambda index: 1000 + index)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setitem(_bevk._entries, "f", lambda *a: seen.append((current[0], a)) or 0)
    _bevk.call_on(0, "f", 1)
    _bevk.call_on(2, "f", 1, 2)
    assert seen == [(0, (1, 1000)), (2, (1, 2, 1002))] and current == [0]
    monkeypatch.setitem(_bevk._entries, "f", lambda *a: 1)
    for index in (0, 1):
        with pytest.raises(RuntimeError):
            _bevk.call_on(index, "f")
