"""Launches of the training-side operators at sizes that they take by their limits: each has fewer
than 2^32 work items, the runtime's limit, and the launches of a kernel have its blocks together."""
import pytest

import _launches

MOST = 2 ** 32 - 1


def _kernels(launches):
    """[(workgroups, threads of each)] of the kernels in a row: launches that go on where the one
    before ended are one kernel's."""
    kernels = []
    for grid, block, first in launches:
        assert grid > 0 and grid * block <= MOST, launches
        if first == 0:
            kernels.append([0, block])
        assert first == kernels[-1][0] and block == kernels[-1][1], launches
        kernels[-1][0] += grid
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
first = lambda k: lambda args: I64.from_address(args[k] + 48).value  # the last member of the geometry
read = first(1)
result = [made("bevk_group_norm_forward", t, P, P, P, t, I64(n), I64(p), c, g, F64(1e-5), 1, P, size(0), P, P, None)]
read = first(2)
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
