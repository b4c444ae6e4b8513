"""linear_cross_entropy's plan: the pieces that a call works in are the ones its
workspace was checked for."""
import os
import subprocess
import sys


from silarray_b200 import _build, _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# getenv as the library sees it: counts the reads of the piece limit.
SHIM = r"""
#define _GNU_SOURCE
#include <dlfcn.h>
#include <string.h>
static int reads;
char *getenv(const char *name) {
  static char *(*real)(const char *);
  if (!real) real = (char *(*)(const char *))dlsym(RTLD_NEXT, "getenv");
  if (strcmp(name, "SILCU_LOSS_PIECE") == 0) reads++;
  return real(name);
}
int loss_piece_reads(void) { return reads; }
"""

# Each entry point once, on shapes that pass every check up to the first one that needs a GPU.
CALLS = r"""
import ctypes as C, importlib.util, sys
spec = importlib.util.spec_from_file_location("_lib", sys.argv[1])
_lib = importlib.util.module_from_spec(spec)
spec.loader.exec_module(_lib)
lib, reads = _lib.lib(), C.CDLL(sys.argv[2]).loss_piece_reads
for dtype in (0, 1):
    a = _lib.CrossEntropyArgs()
    for i, k in enumerate(("dH", "W", "targets", "loss", "lse", "H", "dW")):
        setattr(a, k, (1 << 30) + (i << 28))
    a.rows, a.V, a.D, a.ldh, a.ldw, a.lddh, a.lddw, a.dtype = 300, 5000, 64, 64, 64, 64, 64, dtype
    for f, args in ((lib.silcu_linear_cross_entropy_workspace_bytes, (1,)), (lib.silcu_linear_cross_entropy, (1 << 40, 0, None)),
                    (lib.silcu_linear_cross_entropy_backward, (1 << 40, 0, None))):  # refused: no workspace
        before = reads()
        f(C.byref(a), *args)
        print(f.__name__, reads() - before)
"""


def test_the_piece_limit_is_read_once_per_call(tmp_path):
    """A limit that changes while a call runs cannot part the workspace's check from its use."""
    _build.build()
    (tmp_path / "shim.c").write_text(SHIM)
    shim = tmp_path / "shim.so"
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(shim), str(tmp_path / "shim.c"), "-ldl"], check=True)
    r = subprocess.run([sys.executable, "-c", CALLS, os.path.join(ROOT, "silarray_b200", "_lib.py"), str(shim)],
                       env={**os.environ, "LD_PRELOAD": str(shim)}, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    counts = [line.split() for line in r.stdout.splitlines()]
    assert len(counts) == 6 and all(int(n) <= 1 for _, n in counts), r.stdout
