"""The order in which the two passes of clip_gradients take the tensors, from their launches."""
import pytest

import _launches


@pytest.mark.parametrize("count", [1, 2, 97, 128, 129, 300, 1000])
def test_second_pass_takes_the_same_tables_from_the_last_on(tmp_path, count):
    """A workgroup number within a table stands for the same chunk in both passes, so that the second
    one's kernel can take them from the last to the first on the XCDs that had them; the tables
    themselves come last first. Empty tensors are in none."""
    first, second = _launches.run(tmp_path, f"""
count = {count}
sizes = [0 if k % 5 == 3 else 1 + k * 977 % 30000 for k in range(count)]
at = [(1 + k) << 24 for k in range(count)]
arr = lambda t, v: (t * count)(*v)
V, I = ctypes.c_void_p, ctypes.c_int
def read(name, args):  # addresses, sizes and first chunks of the launch's tensors
    get = lambda t, n, offset: list((t * n).from_address(args[0] + offset))
    n = I.from_address(args[0] + 3844).value
    return name, get(ctypes.c_uint64, n, 0), get(I64, n, 2048), get(I, n + 1, 3072)
tensors = (arr(V, at), arr(I, [0] * count), arr(I64, sizes), arr(V, at), arr(I, [0] * count))
size = I64(lib.bevk_clip_gradients_workspace_bytes(count, tensors[2]))
made("bevk_clip_gradients", count, *tensors, F64(1.0), P, size, P, None)
tables = [l[3] for l in launches]
result = [[t[1:] for t in tables if kernel in t[0]] for kernel in ("squares_kernel", "scale_kernel")]
""")
    sizes = [0 if k % 5 == 3 else 1 + k * 977 % 30000 for k in range(count)]
    assert [(a, n) for at, ns, _ in first for a, n in zip(at, ns)] == [
        ((1 + k) << 24, n) for k, n in enumerate(sizes) if n]
    assert all(len(t[0]) <= 128 for t in first)
    assert second == first[::-1]
