"""The block norm, the 4-bit product and the token scores as a decoder step
uses them together: the norm of a block's output with gate and residual, the
head product of the next norm, the scores of the given tokens. Each step is
checked against float64 from the values the step before stored."""
import ctypes

import numpy as np
import pytest

import test_gpu_block_norm as norm
import test_gpu_q4 as q4
import test_gpu_score as score
from test_gpu_parity import Scope

pytestmark = pytest.mark.gpu


@pytest.fixture
def scope(ctx):
    s = Scope(ctx)
    yield s
    s.close()


class Step:
    """One step over its own buffers."""

    def __init__(self, abi, ctx, scope, rng, dtype, rows, channels=640, columns=1032, classes=1025, k=4):
        self.rows, self.classes, self.k, self.dtype = rows, classes, k, dtype
        self.block = norm.make(rng, dtype, rows, channels, "layer", "row")
        self.head = q4.make(rng, dtype, rows, channels, columns, 64, True, True)
        self.head["scales"] = self.head["scales"] * dtype(4)
        self.tokens = rng.integers(0, classes, rows).astype(np.uint32)
        put = scope.put
        self.buffers = {n: put(self.block[n]) for n in ("input", "gate", "residual", "gamma", "beta", "next_gamma",
                                                       "next_beta")}
        self.output, self.normed = (put(np.zeros((rows, channels), dtype)) for _ in range(2))
        self.logits = put(np.zeros((rows, columns), dtype))
        self.scores = dict(log_probs=put(np.zeros(rows, np.float32)), entropies=put(np.zeros(rows, np.float32)),
                           top_tokens=put(np.zeros((rows, k), np.uint32)),
                           top_log_probs=put(np.zeros((rows, k), np.float32)))
        self.ops = [
            abi.BlockNormOp(ctx, rows=rows, channels=channels, output=self.output, next_output=self.normed,
                            residual_scale=0.5, **self.buffers),
            abi.Q4GemmOp(ctx, a=self.normed, packed=put(abi.pack_q4(self.head["codes"])), scales=put(self.head["scales"]),
                         offsets=put(self.head["offsets"]), bias=put(self.head["bias"]), output=self.logits, rows=rows,
                         inner=channels, columns=columns, group_size=64),
            abi.TokenScoreOp(ctx, logits=self.logits, rows=rows, columns=classes, row_stride=columns,
                             tokens=put(self.tokens), alternatives=k, **self.scores)]

    def enqueue(self, rows=0, stream=None):
        for op in self.ops:
            op.enqueue(rows, stream)

    def feed(self, rng):
        self.block["input"] = rng.standard_normal(self.block["input"].shape).astype(self.dtype)
        self.buffers["input"].upload(self.block["input"])

    def check(self):
        normed, logits = self.normed.download(), self.logits.download()
        norm.check([self.output.download(), normed], self.block)
        q4.check(logits, dict(self.head, a=normed))
        score.check([s.download() for s in self.scores.values()], logits[:, :self.classes], self.tokens, self.k)

    def release(self):
        for op in self.ops:
            op.release()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows", [1, 5, 40, 300])
def test_steps_eager_and_replayed(abi, ctx, scope, dtype, rows):
    rng = np.random.default_rng(rows)
    step = Step(abi, ctx, scope, rng, dtype, rows)
    step.enqueue()
    ctx.synchronize()
    step.check()
    graph = abi.Graph.capture(ctx, ctx.stream)
    with graph:
        step.enqueue(0, ctx.stream)
    for _ in range(3):
        step.feed(rng)
        graph.launch()
        ctx.synchronize()
        step.check()
        step.enqueue(1)  # eager work between the replays
        ctx.synchronize()
    graph.release()
    step.release()


def test_two_streams_at_once(abi, ctx, scope):
    """Two steps of different sizes on two streams, several times over."""
    rng = np.random.default_rng(3)
    steps = [Step(abi, ctx, scope, rng, np.float16, 7), Step(abi, ctx, scope, rng, np.float16, 120)]
    other = ctypes.c_void_p()
    abi.check(abi.load().pk_stream_create(ctx.handle, ctypes.byref(other)))
    for _ in range(5):
        steps[0].enqueue(0, other)
        steps[1].enqueue()
    ctx.synchronize(other)
    ctx.synchronize()
    for step in steps:
        step.check()
        step.release()
    abi.check(abi.load().pk_stream_destroy(ctx.handle, other))


def test_ops_outlive_their_context(abi, scope):
    """An op keeps its context's stream; destroyed ops refuse to run."""
    own = abi.Context(0)
    inner = Scope(own)
    step = Step(abi, own, inner, np.random.default_rng(1), np.float16, 3)
    step.enqueue()
    own.synchronize()
    step.check()
    for op in step.ops:
        op.destroy()
        op.destroy()
        with pytest.raises(abi.PaletteDestroyedError):
            op.enqueue()
    inner.close()
    own.close()
    step.release()


def test_more_rows_than_the_capacity(abi, ctx, scope):
    step = Step(abi, ctx, scope, np.random.default_rng(2), np.float16, 4)
    for op in step.ops:
        with pytest.raises(abi.PaletteRangeError, match=r"active rows must be in \[1, 4\]"):
            op.enqueue(5)
    step.release()
