"""The cache append, the cache attention and the draft verification made on one
GPU while another is current: memory, launches and frees go to the op's own GPU,
and the caller's stays current; an allocation that fails is an error. Runs on the CPU, over the
HIP runtime stub of test_operators_devices.py."""
import os
import shutil
import subprocess
import sys

import pytest

import test_operators_devices as devices

HEAD, TAIL = devices.CHILD.split("makers = [")[0], devices.CHILD.split("for make in makers:", 1)[1]
CHILD = HEAD + """
cache = lambda: dict(rows=4, sequences=2, kv_heads=1, head_dim=64, row_starts=Buffer(12), lengths=Buffer(8),
                     page_table=Buffer(2 * 100 * 4), pages_per_sequence=100, pages=10, page_size=16,
                     key_cache=Buffer(10 * 16 * 64 * 2), value_cache=Buffer(10 * 16 * 64 * 2))
makers = [
    lambda: abi.CacheAppendOp(own, keys=Buffer(512), values=Buffer(512), **cache()),
    lambda: abi.CacheAttentionOp(own, queries=Buffer(1024), output=Buffer(1024), heads=2, **cache()),
    lambda: abi.DraftVerifyOp(own, target=Buffer(4 * 131072 * 2), rows=4, sequences=2, columns=131072,
                              row_starts=Buffer(12), tokens=Buffer(16), uniforms=Buffer(16), draws=Buffer(8),
                              accepted=Buffer(8), next_tokens=Buffer(8))]
for make in makers:""" + TAIL


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc is not installed")
def test_calls_go_to_the_ops_own_device(abi, tmp_path):
    source, stub = tmp_path / "hip_stub.c", tmp_path / "hip_stub.so"
    source.write_text(devices.STUB)
    subprocess.run(["gcc", "-shared", "-fPIC", "-w", str(source), "-o", str(stub)], check=True)
    preload = ":".join(p for p in (str(stub), os.environ.get("LD_PRELOAD")) if p)
    env = dict(os.environ, LD_PRELOAD=preload, PYTHONPATH=devices.ROOT)
    child = subprocess.run([sys.executable, "-c", CHILD, str(stub)], cwd=devices.ROOT, env=env, capture_output=True,
                           text=True, timeout=120)
    assert child.returncode == 0, child.stdout + child.stderr
