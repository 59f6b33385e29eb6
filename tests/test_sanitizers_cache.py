"""The host-side sanitizer leg of the paged cache and the draft verification
(CPU only): their descriptor contracts through the C ABI and through the Node addon."""
import os
import shutil

import pytest

import test_sanitizers as leg


def test_c_abi_contracts():
    lib = leg.build.build_sanitized()
    out = leg.pytest_child("parakeet_wgsl_amd.palette_abi:LIB_PATH", lib,
                           os.path.join(leg.ROOT, "tests", "test_cache_abi_cpu.py"))
    assert " passed" in out


@pytest.mark.skipif(shutil.which("node") is None, reason="node is not installed")
def test_node_addon():
    leg.build.build_sanitized()
    addon = os.path.join(leg.build.SAN, "pk_napi.node")
    if not os.path.exists(addon):
        pytest.skip("Node headers are not installed")
    env = dict(leg.sanitized_env(), PK_NAPI_ADDON=addon)
    out = leg.run_child(["node", os.path.join(leg.ROOT, "tests", "node", "host_cpu_cache.js")], env)
    assert "host_cpu_cache ok" in out
