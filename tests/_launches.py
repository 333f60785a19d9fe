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
static void *module_;
void (*on_kernel)(const void *, const char *);
void (*on_launch)(const void *, unsigned, unsigned, void **);
void **__hipRegisterFatBinary(const void *d) { return &module_; }
void __hipUnregisterFatBinary(void **m) {}
void __hipRegisterVar(void **m, void *v, char *h, char *d, int e, unsigned long s, int c, int g) {}
void __hipRegisterFunction(void **m, const void *f, char *d, const char *name, unsigned t, void *a, void *b,
                           void *c, void *e, int *w) {
  on_kernel(f, name);
}
int __hipPushCallConfiguration(dims g, dims b, unsigned long s, void *st) {
  grid_ = g; block_ = b; shared_ = s; stream_ = st;
  return 0;
}
int __hipPopCallConfiguration(dims *g, dims *b, unsigned long *s, void **st) {
  *g = grid_; *b = block_; *s = shared_; *st = stream_;
  return 0;
}
int hipLaunchKernel(const void *f, dims g, dims b, void **args, unsigned long s, void *st) {
  on_launch(f, g.x, b.x, args);
  return 0;
}
int hipGetLastError(void) { return 0; }
"""

_PRELUDE = r"""
import ctypes, json, sys
shim = ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)
P, I64, F64 = ctypes.c_void_p(0x10000), ctypes.c_int64, ctypes.c_double
kernels, launches = {}, []
read = lambda name, args: None  # what of a launch's arguments is kept
def _on_kernel(f, name):
    kernels[f] = name.decode()
def _on_launch(f, grid, block, args):
    launches.append((kernels[f], grid, block, read(kernels[f], args)))
V, U = ctypes.c_void_p, ctypes.c_uint
_keep = (ctypes.CFUNCTYPE(None, V, ctypes.c_char_p)(_on_kernel),
         ctypes.CFUNCTYPE(None, V, U, U, ctypes.POINTER(V))(_on_launch))
for at, f in zip(("on_kernel", "on_launch"), _keep):
    V.in_dll(shim, at).value = ctypes.cast(f, V).value
lib = ctypes.CDLL(sys.argv[2])
for name in ("group_norm", "embedding_backward", "clip_gradients"):
    getattr(lib, f"bevk_{name}_workspace_bytes").restype = ctypes.c_int64
def made(name, *args):
    "(kernel, workgroups, threads, what was read) of the launches of one call, which has to succeed."
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
