"""Projections whose rows are streamed past a weight in LDS (16 bits, 256 or 512 terms, many rows): every row of the output
and of the gradients against 64 bits, with the bounds of test_gpu_linear.py. The number of rows ends inside a strip, that of
columns inside a part of them; with 512 terms the weight comes in two blocks."""
import pytest
import torch

from test_gpu_linear import DEV, TYPES, _check, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("size", [(50001, 512, 256), (25003, 512, 520), (50001, 256, 512), (30007, 256, 264)], ids=str)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_every_row(size, dtype, act, residual):
    """(50,001 x 256 x 512: without an activation or with ReLU gx is the product of 512 terms, with the others of 1,024.)"""
    t, gy = _inputs(*size, TYPES[dtype], sum(size), residual, device=DEV)
    _check(t, gy, act)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("size", [(50001, 264, 256), (50001, 512, 128)], ids=str)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_gz_in_two_values(size, dtype, act):
    """The gradient of x has twice the output's features as its terms: 512 and 256."""
    t, gy = _inputs(*size, TYPES[dtype], sum(size), False, device=DEV)
    _check(t, gy, act)


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("size", [(40003, 512, 256), (40003, 256, 260)], ids=str)
def test_fp32(size, act, residual):
    """fp32 by a weight in three pieces: streamed for 256 terms, and for 512 with something behind the product."""
    t, gy = _inputs(*size, torch.float32, sum(size), residual, device=DEV)
    _check(t, gy, act)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_non_finite_rows(dtype):
    """A NaN or Inf in a row reaches that row alone, also where a strip's other rows are loaded ahead."""
    from msda_opt2 import linear_act
    t, _ = _inputs(50001, 512, 256, TYPES[dtype], 8, device=DEV)
    good = linear_act(t["x"], t["weight"], t["bias"], "relu", t["residual"])
    x = t["x"].clone()
    rows = torch.tensor([0, 15, 16, 2049, 50000], device=DEV)
    for bad in (float("nan"), float("inf")):
        x[rows, 300] = bad
        y = linear_act(x, t["weight"], t["bias"], "relu", t["residual"])
        keep = torch.ones(50001, dtype=torch.bool, device=DEV)
        keep[rows] = False
        assert torch.equal(y[keep], good[keep]) and not torch.equal(y[rows], good[rows])
