"""The block norm, the 4-bit product and the token scores made on one GPU while
another is current: memory, launches and frees go to the op's own GPU, and the
caller's stays current. Runs on the CPU: a child process loads the library
with a HIP runtime stub of eight devices that notes where calls go."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

STUB = r"""
#include <stdlib.h>
static int current;
int stub_calls, stub_wrong, stub_fail_malloc;
static void on_own(void) { ++stub_calls; stub_wrong += current != 3; }
int hipGetDeviceCount(int* n) { *n = 8; return 0; }
int hipSetDevice(int d) { current = d; return 0; }
int hipGetDevice(int* d) { *d = current; return 0; }
int hipStreamCreateWithFlags(void** s, unsigned f) { *s = malloc(1); return 0; }
int hipStreamDestroy(void* s) { return 0; }
int hipStreamSynchronize(void* s) { return 0; }
int hipStreamIsCapturing(void* s, int* status) { *status = 0; return 0; }
int hipDeviceSynchronize(void) { on_own(); return 0; }
int hipGetLastError(void) { return 0; }
int hipMalloc(void** p, size_t n) { on_own(); *p = stub_fail_malloc ? 0 : malloc(64); return stub_fail_malloc ? 2 : 0; }
int hipFree(void* p) { on_own(); free(p); return 0; }
typedef struct { unsigned x, y, z; } dim;
int hipLaunchKernel(const void* f, dim grid, dim block, void** args, size_t lds, void* stream) { on_own(); return 0; }
int __hipPushCallConfiguration(dim g, dim b, size_t lds, void* s) { return 0; }
int __hipPopCallConfiguration(dim* g, dim* b, size_t* lds, void** s) { return 0; }
"""

CHILD = """
import ctypes, sys
stub = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
import numpy as np
import parakeet_wgsl_amd.palette_abi as abi
class Buffer:
    at = 1 << 20
    def __init__(self, nbytes, dtype=np.float16):
        Buffer.at += 1 << 30
        self.ptr, self.nbytes, self.dtype = Buffer.at, nbytes, np.dtype(dtype)
value = lambda name: ctypes.c_int.in_dll(stub, name).value
def current():
    d = ctypes.c_int()
    stub.hipGetDevice(ctypes.byref(d))
    return d.value
own = abi.Context(3)
stub.hipSetDevice(5)
makers = [
    lambda: abi.BlockNormOp(own, rows=4, channels=64, input=Buffer(512), output=Buffer(512)),
    lambda: abi.Q4GemmOp(own, a=Buffer(512), packed=Buffer(64 * 64 // 2), scales=Buffer(2 * 64 * 2), output=Buffer(512),
                         rows=4, inner=64, columns=64, group_size=32),
    lambda: abi.TokenScoreOp(own, logits=Buffer(2 * 131072 * 2), rows=2, columns=131072, entropies=Buffer(8))]
for make in makers:
    before = value("stub_calls")
    op = make()
    op.enqueue()
    assert value("stub_calls") > before and current() == 5, (value("stub_calls"), current())
    op.release()
    assert current() == 5
for make in makers[1:]:  # those that allocate
    ctypes.c_int.in_dll(stub, "stub_fail_malloc").value = 1
    try:
        make()
        raise SystemExit("an allocation that fails is an error")
    except abi.PaletteError as e:
        assert e.status == abi.ALLOCATION_FAILURE and "cannot allocate" in str(e), e
    ctypes.c_int.in_dll(stub, "stub_fail_malloc").value = 0
    assert current() == 5
print("wrong", value("stub_wrong"), "of", value("stub_calls"))
assert not value("stub_wrong")
"""


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc is not installed")
def test_calls_go_to_the_ops_own_device(abi, tmp_path):
    source, stub = tmp_path / "hip_stub.c", tmp_path / "hip_stub.so"
    source.write_text(STUB)
    subprocess.run(["gcc", "-shared", "-fPIC", "-w", str(source), "-o", str(stub)], check=True)
    preload = ":".join(p for p in (str(stub), os.environ.get("LD_PRELOAD")) if p)
    env = dict(os.environ, LD_PRELOAD=preload, PYTHONPATH=ROOT)
    child = subprocess.run([sys.executable, "-c", CHILD, str(stub)], cwd=ROOT, env=env, capture_output=True, text=True,
                           timeout=120)
    assert child.returncode == 0, child.stdout + child.stderr
