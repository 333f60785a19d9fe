"""The kernel launches of libbevk.so's entry points, recorded instead of made, so that a grid and
its arguments can be tested without a GPU and at sizes that no tensor here has: a process of its
own loads stand-ins for the runtime's launch functions ahead of the library."""
import json
import subprocess
import sys

_STAND_INS = r"""
typedef struct { unsigned x, y, z; } dims;
static dims grid_, block_;
static unsigned long shared_;
static void *stream_;
void (*on_launch)(unsigned, unsigned, void **);
int __hipPushCallConfiguration(dims g, dims b, unsigned long s, void *st) {
  grid_ = g; block_ = b; shared_ = s; stream_ = st;
  return 0;
}
int __hipPopCallConfiguration(dims *g, dims *b, unsigned long *s, void **st) {
  *g = grid_; *b = block_; *s = shared_; *st = stream_;
  return 0;
}
int hipLaunchKernel(const void *f, dims g, dims b, void **args, unsigned long s, void *st) {
  on_launch(g.x, b.x, args);
  return 0;
}
int hipGetLastError(void) { return 0; }
"""

_PRELUDE = r"""
import ctypes, json, sys
shim = ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
P, I64, F64 = ctypes.c_void_p(0x10000), ctypes.c_int64, ctypes.c_double
for name in ("group_norm", "embedding_backward", "clip_gradients"):
    getattr(lib, f"bevk_{name}_workspace_bytes").restype = ctypes.c_int64
launches = []
read = lambda args: None  # what of a launch's arguments is kept
def _launch(grid, block, args):
    launches.append((grid, block, read(args)))
_keep = ctypes.CFUNCTYPE(None, ctypes.c_uint, ctypes.c_uint, ctypes.POINTER(ctypes.c_void_p))(_launch)
ctypes.c_void_p.in_dll(shim, "on_launch").value = ctypes.cast(_keep, ctypes.c_void_p).value
def made(name, *args):
    "The launches of one call, which has to succeed."
    launches.clear()
    assert getattr(lib, name)(*args) == 0, name
    return list(launches)
"""


def run(tmp_path, body):
    """What `body` leaves in `result` (JSON), run with `made` and `read` of the prelude."""
    import _bevk
    source, shim = tmp_path / "stand_ins.c", tmp_path / "stand_ins.so"
    source.write_text(_STAND_INS)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", str(source), "-o", str(shim)], check=True)
    code = _PRELUDE + body + "\nprint(json.dumps(result))"
    done = subprocess.run([sys.executable, "-c", code, str(shim), _bevk.library_path()],
                          capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stderr
    return json.loads(done.stdout)
