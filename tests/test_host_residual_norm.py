"""Refusals of the residual norm on the CPU, in Python and at the C ABI: nothing here reaches a launch
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
    x = torch.zeros(2, 3, 8)
    with pytest.raises(RuntimeError, match="HIP"):
        msda_opt2.residual_norm(x)
    with torch.no_grad(), pytest.raises(RuntimeError, match="HIP"):
        msda_opt2.residual_norm(x, x)


@pytest.mark.parametrize("kw,code,match", [
    (dict(dtype=3), UNSUPPORTED, "Double"), (dict(pd=3), UNSUPPORTED, "Double"), (dict(gd=9), UNSUPPORTED, "unknown"),
    (dict(dtype=1, pd=2, gd=1), INVALID, "input's type"), (dict(dtype=1, pd=1, gd=2), INVALID, "input's type"),
    (dict(rows=0), INVALID, "positive"), (dict(c=0), INVALID, "positive"), (dict(rows=-4), INVALID, "positive"),
    (dict(sr=-1), INVALID, "positive"), (dict(sr=3), INVALID, "whole sets"), (dict(kind=2), INVALID, "kind"),
    (dict(rows=2 ** 38), INVALID, "2\\^40"), (dict(c=2 ** 30 + 1), INVALID, "2\\^30")])
def test_refusals(kw, code, match):
    lib = _bevk.lib()

    def forward(dtype=0, pd=0, gd=0, rows=4, sr=0, c=8, kind=0):
        return lib.bevk_residual_norm_forward(dtype, P, P, None, None, None, None, None, pd, gd, rows, sr, c, kind, 0,
                                              1.0, 1e-5, P, P, P, None)

    def backward(dtype=0, pd=0, gd=0, rows=4, sr=0, c=8, kind=0):
        return lib.bevk_residual_norm_backward(dtype, P, None, P, P, P, None, None, None, None, pd, gd, rows, sr, c,
                                               kind, 0, 1.0, P, 1 << 40, P, P, None, None, None, None, None, None)
    for f in (forward, backward):
        assert f(**kw) == code and re.search(match, _err()), _err()


def test_pointers_and_workspace():
    lib = _bevk.lib()
    size = lib.bevk_residual_norm_backward_workspace_bytes
    assert size(0, 4, 0, 8) > 0 and size(3, 4, 0, 8) == -1 and size(0, 0, 0, 8) == -1 and size(0, 5, 2, 8) == -1

    def forward(x=P, y=P, eps=1e-5):
        return lib.bevk_residual_norm_forward(0, x, None, None, None, None, None, None, 0, 0, 4, 0, 8, 0, 0, 1.0, eps,
                                              y, None, None, None)

    assert forward(x=None) == INVALID and "null" in _err()
    assert forward(y=None) == INVALID and "null" in _err()
    assert forward(eps=-1.0) == INVALID and "eps" in _err()
    assert forward(eps=float("nan")) == INVALID and "eps" in _err()

    def backward(gy=P, x=P, st=P, block=0, ws=P, wb=1 << 20, gg=None, gbw=None):
        return lib.bevk_residual_norm_backward(0, gy, None, x, None, st, None, None, None, None, 0, 0, 4, 0, 8, 0, block,
                                               1.0, ws, wb, P, P, None, None, gg, gbw, None, None)
    for kw in (dict(gy=None), dict(st=None), dict(x=None), dict(x=None, block=1), dict(ws=None)):
        assert backward(**kw) == INVALID and "null" in _err()
    assert backward(wb=16) == INVALID and "too small" in _err()
    assert backward(ws=P + 8) == INVALID and "16-byte" in _err()
    assert backward(gbw=P) == INVALID and "block norm" in _err()
