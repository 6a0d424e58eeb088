"""What swb_create says and leaves behind where one of its steps fails: the CUDA runtime's calls are answered by a stand-in."""
import os
import shutil
import subprocess
import sys

import pytest

from sparsewave_b200 import _lib
from sparsewave_b200.build import LIB, ROOT

# Each call succeeds, but for the one named in FAILS; memory handed out and taken back is counted.
STAND_IN = r"""
#include <cstdlib>
#include <cstring>
namespace {
int pending = 0, held = 0, pools = 0;
int answer(const char *name) {
  const char *fails = getenv("FAILS");
  if (fails && !strcmp(fails, name)) return pending = 2;  // cudaErrorMemoryAllocation
  return 0;
}
}
extern "C" {
int cudaGetDeviceCount(int *n) { *n = 1; return answer("cudaGetDeviceCount"); }
int cudaSetDevice(int) { return answer("cudaSetDevice"); }
int cudaDeviceGetAttribute(int *v, int, int) { *v = 148; return 0; }
int cudaMalloc(void **p, size_t) { int e = answer("cudaMalloc"); if (!e) { *p = &held; ++held; } return e; }
int cudaFree(void *p) { if (p) --held; return 0; }
int cudaMemset(void *, int, size_t) { return answer("cudaMemset"); }
int cudaMemPoolCreate(void **p, const void *) { int e = answer("cudaMemPoolCreate"); if (!e) { *p = &pools; ++pools; } return e; }
int cudaMemPoolDestroy(void *) { --pools; return 0; }
int cudaMemPoolSetAttribute(void *, int, void *) { return answer("cudaMemPoolSetAttribute"); }
int cudaGetLastError() { int e = pending; pending = 0; return e; }
int stand_in_pending() { return pending; }
int stand_in_held() { return held + pools; }
}
"""

PROGRAM = """
import ctypes as C, sys
lib, fake = C.CDLL(sys.argv[1]), C.CDLL(None)
lib.swb_last_error.restype = C.c_char_p
lib.swb_last_error.argtypes = [C.c_void_p]
ctx = C.c_void_p()
st = lib.swb_create(C.byref(ctx), 0)
print(st, bool(ctx.value), fake.stand_in_pending(), fake.stand_in_held(), lib.swb_last_error(None).decode(), sep="|")
"""


@pytest.fixture(scope="module")
def created(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    folder = tmp_path_factory.mktemp("create")
    (folder / "stand_in.cpp").write_text(STAND_IN)
    subprocess.run(["g++", "-shared", "-fPIC", str(folder / "stand_in.cpp"), "-o", str(folder / "stand_in.so")], check=True)
    import torch  # the runtime that the library is loaded with
    runtime = os.path.join(os.path.dirname(os.path.dirname(torch.__file__)), "nvidia", "cuda_runtime", "lib")

    def run(fails):
        paths = ":".join(filter(None, [runtime, os.environ.get("LD_LIBRARY_PATH")]))
        out = subprocess.run([sys.executable, "-c", PROGRAM, str(LIB)], check=True, capture_output=True, text=True, cwd=ROOT,
                             env={**os.environ, "LD_PRELOAD": str(folder / "stand_in.so"), "FAILS": fails, "LD_LIBRARY_PATH": paths}).stdout
        st, made, pending, held, message = out.strip().split("|")
        return int(st), made == "True", int(pending), int(held), message

    return run


def test_success(created):
    st, made, pending, held, _ = created("")
    assert (st, made, pending, held) == (_lib.SWB_OK, True, 0, 2)


@pytest.mark.parametrize("call", ["cudaGetDeviceCount", "cudaSetDevice", "cudaMalloc", "cudaMemset", "cudaMemPoolCreate", "cudaMemPoolSetAttribute"])
def test_a_step_that_fails(created, call):
    """The message names the step, the error is not left pending, and nothing stays allocated."""
    st, made, pending, held, message = created(call)
    assert (st, made, pending, held) == (_lib.SWB_ERR_CUDA, False, 0, 0)
    assert call in message
