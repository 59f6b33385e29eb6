"""The block norm, the 4-bit product and the token scores on HIP's default
stream, by its legacy handle: in order with the copies before and after them,
with nothing waited for between."""
import numpy as np
import pytest

import test_gpu_operators as operators
from test_gpu_parity import Scope

pytestmark = pytest.mark.gpu

DEFAULT = 1  # hipStreamLegacy


def test_steps_in_order_on_the_default_stream(abi, ctx):
    rng = np.random.default_rng(9)
    scope = Scope(ctx)
    step = operators.Step(abi, ctx, scope, rng, np.float16, 40)
    results = [step.output, step.normed, step.logits, *step.scores.values()]
    inputs, expected = [], []
    for _ in range(2):
        step.feed(rng)
        step.enqueue()
        ctx.synchronize()
        step.check()
        inputs.append(scope.put(step.block["input"]))
        expected.append([r.download() for r in results])
    long = [scope.empty(1 << 28, np.uint8) for _ in range(2)]
    copies = [[scope.empty(r.shape, r.dtype) for r in results] for _ in range(6)]
    for i, kept in enumerate(copies):
        for _ in range(4):
            ctx.copy(long[i % 2], long[1 - i % 2], DEFAULT)  # the step's input waits behind these
        ctx.copy(step.buffers["input"], inputs[i % 2], DEFAULT)
        step.enqueue(0, DEFAULT)
        for to, result in zip(kept, results):
            ctx.copy(to, result, DEFAULT)
    ctx.synchronize(DEFAULT)
    for i, kept in enumerate(copies):
        for got, want in zip(kept, expected[i % 2]):
            np.testing.assert_array_equal(got.download(), want)
    step.release()
    scope.close()
