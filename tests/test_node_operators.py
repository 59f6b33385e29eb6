"""The block norm, the 4-bit product and the token scores through the Node
host: contracts on the CPU, and all three in one command buffer on the GPU,
each step against float64 from the values the step before stored."""
import json

import numpy as np
import pytest

import test_gpu_block_norm as norm
import test_gpu_q4 as q4
import test_gpu_score as score
from test_node_host import needs_node, run_node


@needs_node
def test_contracts_on_cpu():
    assert "host_cpu_operators ok" in run_node("host_cpu_operators.js")


@needs_node
@pytest.mark.gpu
def test_one_command_buffer(tmp_path, abi):
    rng = np.random.default_rng(12)
    rows, channels, columns, classes, group, alternatives, active = 20, 640, 1032, 1025, 64, 4, 17
    block = norm.make(rng, np.float16, rows, channels, "rms", "all", beta=False)
    head = q4.make(rng, np.float16, rows, channels, columns, group, bias=True)
    tokens = rng.integers(0, classes, rows).astype(np.uint32)
    arrays = dict(input=block["input"], residual=block["residual"], gate=block["gate"], gamma=block["gamma"],
                  nextGamma=block["next_gamma"], packed=abi.pack_q4(head["codes"]), scales=head["scales"],
                  bias=head["bias"], tokens=tokens)
    spec = dict(rows=rows, channels=channels, columns=columns, classes=classes, groupSize=group,
                alternatives=alternatives, active=active, directory=str(tmp_path))
    for name, a in arrays.items():
        spec[name] = str(tmp_path / f"{name}.bin")
        np.ascontiguousarray(a).tofile(spec[name])
    (tmp_path / "case.json").write_text(json.dumps(spec))
    assert "host_gpu_operators ok" in run_node("host_gpu_operators.js", str(tmp_path / "case.json"))

    def got(name, dtype, *shape):
        return np.fromfile(tmp_path / f"{name}.out", dtype).reshape(shape)
    normed = got("normed", np.float16, rows, channels)
    norm.check([got("output", np.float16, rows, channels), normed], block, rows=active)
    head["a"] = normed
    logits = got("logits", np.float16, rows, columns)
    q4.check(logits, head, rows=active)
    score.check([got("logProbs", np.float32, rows), got("entropies", np.float32, rows),
                 got("topTokens", np.uint32, rows, alternatives), got("topLogProbs", np.float32, rows, alternatives)],
                logits[:, :classes], tokens, alternatives, rows=active)
