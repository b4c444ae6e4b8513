"""linear_cross_entropy's plan: the pieces that a call works in are the ones its
workspace was checked for."""
import ctypes as C
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


def args(**kw):
    a = _lib.CrossEntropyArgs()
    for i, k in enumerate(("dH", "W", "targets", "loss", "lse", "H", "dW")):
        setattr(a, k, (i + 1) << 34)
    a.rows, a.V, a.D = 4096, 1 << 17, 768
    for k, v in kw.items():
        setattr(a, k, v)
    for k in ("ldh", "ldw", "lddh", "lddw"):
        setattr(a, k, getattr(a, k) or a.D)
    return a


def test_what_the_workspace_grows_with():
    """Of the vocabulary only the forward's parts: two of 8 bytes for a tile of 256 columns (for 16
    at least, where few rows have narrow tiles).  Pieces of about the same size hold the rest."""
    _build.build()
    size = _lib.lib().silcu_linear_cross_entropy_workspace_bytes
    vocabularies = [1 << 17, 1 << 18, 1 << 20]
    for rows in (1024, 4096):
        parts = [16 * rows * v // 256 for v in vocabularies]
        bf16, f32 = ([[size(C.byref(args(rows=rows, V=v, dtype=d)), b) for v in vocabularies] for b in (0, 1)] for d in (1, 0))
        for s, n in zip(bf16[0], parts):  # its operands are read in place
            assert abs((s - bf16[0][0]) - (n - parts[0])) <= n // 32, rows
        for sizes in (bf16[1], *f32):
            for s, n in zip(sizes, parts):
                assert s <= 1.5 * sizes[0] + 1.1 * n, rows


def test_the_workspace_of_another_layout():
    """A query holds for operands laid out as they are in the call: unaligned ones are copied."""
    _build.build()
    lib = _lib.lib()
    aligned = args(dtype=1)
    for kw in (dict(H=(6 << 34) + 2), dict(W=(2 << 34) + 2), dict(ldw=769), dict(ldh=769)):
        other = args(dtype=1, **kw)
        for f, backward in ((lib.silcu_linear_cross_entropy, 0), (lib.silcu_linear_cross_entropy_backward, 1)):
            need, own = (lib.silcu_linear_cross_entropy_workspace_bytes(C.byref(a), backward) for a in (aligned, other))
            assert own >= need
            if own > need:
                assert f(C.byref(other), C.c_void_p(1 << 40), need, None) == 4
            assert f(C.byref(other), C.c_void_p(1 << 40), own - 1, None) in (4, 2)
