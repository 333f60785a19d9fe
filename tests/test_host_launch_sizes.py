"""Launches of the training-side operators at sizes that they take by their limits: each has fewer
than 2^32 work items, the runtime's limit, and the launches of a kernel have its blocks together."""
import pytest

import _launches

MOST = 2 ** 32 - 1


def _kernels(launches):
    """[(workgroups, threads of each)] of the kernels in a row: launches of one kernel, each from where
    the one before ended."""
    kernels, before = [], None
    for name, grid, block, first in launches:
        assert grid > 0 and grid * block <= MOST, launches
        if name != before:
            kernels.append([0, block])
        assert first == kernels[-1][0], launches
        kernels[-1][0] += grid
        before = name
    return [tuple(k) for k in kernels]


# (batch, pixels, channels, groups); tiles: 128 bytes of channels (or 64 single ones) by at most 64
# rounds of positions
NORMS = [(131072, 1, 1024, 32), (263168, 1, 1024, 32), (1 << 24, 1, 64, 8), (1, 1 << 33, 1, 1),
         (1 << 22, 3, 40, 8), (1 << 25, 2, 65, 5), (3, 1, 1 << 30, 1)]


@pytest.mark.parametrize("dtype", [0, 2], ids=["fp32", "bf16"])
@pytest.mark.parametrize("sizes", NORMS, ids=str)
def test_group_norm(tmp_path, sizes, dtype):
    n, p, c, g = sizes
    forward, backward = _launches.run(tmp_path, f"""
n, p, c, g, t = {n}, {p}, {c}, {g}, {dtype}
size = lambda back: I64(lib.bevk_group_norm_workspace_bytes(t, back, I64(n), I64(p), c, g, 1))
def read(name, args):  # the last member of the geometry
    return I64.from_address(args[2 if "grad" in name else 1] + 48).value
result = [made("bevk_group_norm_forward", t, P, P, P, t, I64(n), I64(p), c, g, F64(1e-5), 1, P, size(0), P, P, None)]
result += [made("bevk_group_norm_backward", t, P, P, P, P, t, I64(n), I64(p), c, g, 1, P, P, size(1), P, P, P, None)]
""")
    wide = c * (4, 2, 2)[dtype] % 16 == 0
    slab, rows = (128 // (4, 2, 2)[dtype], 32) if wide else (64, 4)
    slabs = -(-c // slab)
    each = 64 * rows  # (far more tiles than the least wanted, or one for each image)
    tiles = n * slabs * -(-p // each)
    back = -(-tiles // 8) * 8
    forward, (sums, (values, _)) = _kernels(forward), _kernels(backward)
    if forward[0][1] == 1024:
        assert forward == [(n * slabs, 1024)]
    else:
        assert forward == [(tiles, 256), (back, 256)]
    assert sums == (tiles, 256) and values - back in range(-(-c // 32), -(-c // 32) + 8)


# (n, rows, dim)
LOOKUPS = [((1 << 31) - 1024, 7, 9), ((1 << 31) - 1024, 1000, 1), (1000, (1 << 30) + 5, 1),
           (5, (1 << 31) - 256, 8), (1 << 24, 100, 2049), ((1 << 28) + 100, 131072, 1), (1 << 29, 3, 64)]


@pytest.mark.parametrize("dtype", [0, 1], ids=["fp32", "fp16"])
@pytest.mark.parametrize("sizes", LOOKUPS, ids=str)
def test_embedding(tmp_path, sizes, dtype):
    n, rows, dim = sizes
    forward, backward = _launches.run(tmp_path, f"""
n, rows, dim, t = {n}, {rows}, {dim}, {dtype}
size = I64(lib.bevk_embedding_backward_workspace_bytes(t, I64(n), I64(rows), dim))
one = ctypes.c_float(1.0)
def read(name, args):  # the lookup's own argument, a member of the others' sizes
    at = (args[5] if "lookup" in name else args[1] + 20 if "sort" in name else
          args[2 if "sum" in name else 1] + 28)
    return (I64 if "lookup" in name else ctypes.c_int).from_address(at).value
result = [made("bevk_embedding_forward", t, P, I64(rows), dim, P, 0, I64(n), one, P, None),
          made("bevk_embedding_backward", t, P, P, 0, I64(n), I64(rows), dim, one, I64(-1), P, size, P, None)]
""")
    vector = next(v for v in (16 // (4, 2)[dtype], 8 // (4, 2)[dtype], 1) if dim % v == 0)
    assert _kernels(forward) == [(-(-n * dim // vector // 1024), 256)]
    owners = 256
    while -(-rows // owners) > 512:
        owners *= 2
    lanes = 1
    while lanes < 64 and lanes * vector < dim:
        lanes *= 2
    slices = -(-dim // (lanes * vector))
    chunks = -(-n // 32) * slices if n > 32 else 0
    own = min(1 << 20, -(-rows * slices // (256 // lanes)))
    assert _kernels(backward) == [(owners, 1024), (chunks + own, 256)] + [(chunks, 256)] * (chunks > 0)


def test_embedding_refuses_more_than_2_40_values():
    import ctypes

    import _bevk
    lib, P = _bevk.lib(), ctypes.c_void_p(0x10000)
    for n, rows, dim in ((1 << 30, 5, 1025), (5, 1 << 30, 1025)):
        assert lib.bevk_embedding_forward(0, P, rows, dim, P, 0, n, 1.0, P, None) == 1
        assert "2^40" in lib.bevk_last_error().decode()
        assert lib.bevk_embedding_backward_workspace_bytes(0, n, rows, dim) == -1
        assert lib.bevk_embedding_backward(0, P, P, 0, n, rows, dim, 1.0, -1, P, 1 << 50, P, None) == 1
