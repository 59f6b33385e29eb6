"""The cache append, the cache attention and the draft verification through the Node
host: contracts on the CPU, and all three in one command buffer on the GPU."""
import json

import numpy as np
import pytest

import test_gpu_cache as cache_test
import test_gpu_verify as verify
from test_node_host import needs_node, run_node


@needs_node
def test_contracts_on_cpu():
    assert "host_cpu_cache ok" in run_node("host_cpu_cache.js")


@needs_node
@pytest.mark.gpu
def test_one_command_buffer(tmp_path):
    rng = np.random.default_rng(21)
    heads, kv_heads, dim, columns, active = 4, 2, 64, 900, 3
    cache = cache_test.Cache(rng, np.float16, [4, 2, 7, 3], [30, 100, 7, 50], kv_heads, dim, 16)
    rows = cache.rows
    case = verify.make(rng, np.float16, cache.counts, columns, temperature=0.75)
    q, k, v = (rng.standard_normal((rows, n * dim)).astype(np.float16) for n in (heads, kv_heads, kv_heads))
    frequencies = (100.0 ** (-np.arange(dim // 2) / (dim // 2))).astype(np.float32)
    arrays = dict(queries=q, keys=k, values=v, frequencies=frequencies, rowStarts=cache.starts, lengths=cache.lengths,
                  pageTable=cache.table, keyCache=cache.keys, valueCache=cache.values, target=case["target"],
                  draft=case["draft"], tokens=case["tokens"], uniforms=case["uniforms"], draws=case["draws"])
    files = {}
    for name, a in arrays.items():
        files[name] = str(tmp_path / f"{name}.bin")
        np.ascontiguousarray(a).tofile(files[name])
    spec = dict(files=files, rows=rows, sequences=cache.sequences, heads=heads, kvHeads=kv_heads, headDim=dim,
                columns=columns, active=active, directory=str(tmp_path),
                cache=dict(pagesPerSequence=cache.width, pages=cache.pages, pageSize=16))
    (tmp_path / "case.json").write_text(json.dumps(spec))
    assert "host_gpu_cache ok" in run_node("host_gpu_cache.js", str(tmp_path / "case.json"))

    def got(name, dtype):
        return np.fromfile(tmp_path / f"{name}.out", dtype)
    rotated = got("rotated", np.float16).reshape(rows, -1)
    stored = [rotated, got("keyCache", np.float16), got("valueCache", np.float16)]
    cache_test.check_append(cache, stored, q, k, v, frequencies, "neighbours", heads=heads, active=active)
    cache.keys, cache.values = stored[1:]
    cache_test.check_attention(cache, got("attended", np.float16), rotated, heads, active=active, cap=20.0, window=60)
    margins = []
    want = verify.formula(case["target"], case["draft"], case["tokens"], case["starts"], case["uniforms"], case["draws"], 0.75,
                          False, margins)
    assert min(margins) > verify.MARGIN
    np.testing.assert_array_equal(got("accepted", np.uint32)[:active], want[0][:active])
    np.testing.assert_array_equal(got("nextTokens", np.uint32)[:active], want[1][:active])
