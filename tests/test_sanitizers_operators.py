"""The host-side sanitizer leg of the block norm, the 4-bit product and the
token scores (CPU only): their descriptor contracts through the C ABI and
through the Node addon."""
import os
import shutil

import pytest

import test_sanitizers as leg


@pytest.mark.parametrize("name", ["test_operators_abi_cpu.py", "test_operators_overlap.py"])
def test_c_abi_contracts(name):
    lib = leg.build.build_sanitized()
    out = leg.pytest_child("parakeet_wgsl_amd.palette_abi:LIB_PATH", lib, os.path.join(leg.ROOT, "tests", name))
    assert " passed" in out


@pytest.mark.skipif(shutil.which("node") is None, reason="node is not installed")
@pytest.mark.parametrize("name", ["host_cpu_operators", "host_cpu_operator_fields"])
def test_node_addon(name):
    leg.build.build_sanitized()
    addon = os.path.join(leg.build.SAN, "pk_napi.node")
    if not os.path.exists(addon):
        pytest.skip("Node headers are not installed")
    env = dict(leg.sanitized_env(), PK_NAPI_ADDON=addon)
    out = leg.run_child(["node", os.path.join(leg.ROOT, "tests", "node", name + ".js")], env)
    assert f"{name} ok" in out
