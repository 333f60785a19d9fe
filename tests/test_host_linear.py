"""Refusals of the projections on the CPU, in Python and at the C ABI: nothing here reaches a launch
(fake device addresses are never followed)."""
import re

import pytest
import torch

import _bevk
import msda_opt2

INVALID, UNSUPPORTED = 1, 2
P = 0x10000


def _err():
    return _bevk.lib().bevk_last_error().decode()


def test_needs_a_device():
    x, w = torch.zeros(2, 3, 8), torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="HIP"):
        msda_opt2.linear_act(x, w)
    with torch.no_grad(), pytest.raises(RuntimeError, match="HIP"):
        msda_opt2.linear_act(x, w)


@pytest.mark.parametrize("kw,code,match", [
    (dict(dtype=3), UNSUPPORTED, "Double"), (dict(bd=9), UNSUPPORTED, "unknown"),
    (dict(dtype=1, bd=2), INVALID, "input's type"), (dict(rows=0), INVALID, "positive"),
    (dict(k=0), INVALID, "positive"), (dict(n=-1), INVALID, "positive"), (dict(k=2 ** 24 + 1), INVALID, "2\\^24"),
    (dict(rows=2 ** 31), INVALID, "2\\^31"), (dict(rows=2 ** 30, n=2 ** 12), INVALID, "2\\^40"),
    (dict(k=2 ** 21, n=2 ** 20), INVALID, "2\\^40"), (dict(act=4), INVALID, "activation"),
    (dict(act=-1), INVALID, "activation"), (dict(x=None), INVALID, "null"), (dict(w=None), INVALID, "null"),
    (dict(y=None), INVALID, "null")])
def test_refusals(kw, code, match):
    lib = _bevk.lib()

    def forward(dtype=0, x=P, w=P, bd=0, rows=4, k=8, n=8, act=0, y=P):
        return lib.bevk_linear_forward(dtype, x, w, None, bd, None, rows, k, n, act, P, 1 << 50, y, None, None)

    def backward(dtype=0, x=P, w=P, bd=0, rows=4, k=8, n=8, act=0, y=P):
        return lib.bevk_linear_backward(dtype, y, x, w, P, rows, k, n, act, bd, P, 1 << 50, P, P, P, None)
    for f in (forward, backward):
        assert f(**kw) == code and re.search(match, _err()), _err()


def test_workspace():
    lib = _bevk.lib()
    size = lib.bevk_linear_workspace_bytes
    assert size(0, 0, 0, 4, 8, 8, 0) >= 0 and size(3, 0, 0, 4, 8, 8, 0) == -1 and size(0, 1, 0, 0, 8, 8, 0) == -1
    # operands on 16-byte boundaries: none for rows that are loaded as they are, some off them for a split sum
    assert size(1, 0, 1, 4, 2048, 64, 0) == 0 < size(1, 0, 0, 4, 2048, 64, 0)
    need = size(1, 1, 0, 4000, 256, 256, 3)
    assert need >= 4000 * 256 * 2

    def backward(z=P, ws=P, wb=1 << 50):
        return lib.bevk_linear_backward(1, P, P, P, z, 4000, 256, 256, 3, 1, ws, wb, P, P, P, None)
    assert backward(z=None) == INVALID and "null" in _err()
    assert backward(ws=None) == INVALID and "null" in _err()
    assert backward(wb=need - 1) == INVALID and "too small" in _err()
    assert backward(ws=P + 8) == INVALID and "16-byte" in _err()
