"""Group norm's backward: where its second launch's tiles begin among the workgroups."""
import pytest

import _launches


@pytest.mark.parametrize("channels", [8, 64, 75, 96, 100, 128, 256, 320, 512, 1000])
def test_tiles_begin_at_a_multiple_of_the_xcds(tmp_path, channels):
    """A workgroup runs on the XCD that its number modulo 8 says. The tiles come behind the workgroups
    of the parameters' gradients, and each on the XCD that had it in the first launch only if those
    are a multiple of 8."""
    result = _launches.run(tmp_path, f"""
c = {channels}
def read(name, args):
    return name, ctypes.c_int.from_address(args[4]).value if "grad_x" in name else None
size = I64(lib.bevk_group_norm_workspace_bytes(2, 1, I64(6), I64(5800), c, 1, 1))
result = made("bevk_group_norm_backward", 2, P, P, P, P, 2, I64(6), I64(5800), c, 1, 1, P, P, size, P, P, P, None)
""")
    (_, tiles, _, _), (_, workgroups, _, (name, before)) = result
    assert "grad_x_kernel" in name and before % 8 == 0 and before >= channels / 32
    assert workgroups == before + -(-tiles // 8) * 8
