"""The cache append, the cache attention, the 4-bit head product and the draft
verification as a decoder uses them together: several steps of drafts over a cache
that grows, eager, on two streams and replayed from a graph. Each stage is
checked against float64 from the values that the stage before stored."""
import ctypes

import numpy as np
import pytest

import test_gpu_cache as cache_test
import test_gpu_q4 as q4
import test_gpu_verify as verify
from test_gpu_parity import Scope

pytestmark = pytest.mark.gpu


@pytest.fixture
def scope(ctx):
    s = Scope(ctx)
    yield s
    s.close()


class Decoder:
    """Sequences that grow by the rows of each step, over their own buffers."""

    def __init__(self, abi, ctx, scope, rng, dtype, counts, lengths, heads=4, kv_heads=2, dim=64, page=16, columns=130,
                 most=400, window=0):
        self.ctx, self.rng, self.dtype, self.heads, self.window = ctx, rng, dtype, heads, window
        self.cache = c = cache_test.Cache(rng, dtype, counts, [most] * len(counts), kv_heads, dim, page)
        c.lengths = np.array(lengths, np.uint32)
        rows, self.row = c.rows, (heads + 2 * kv_heads) * dim
        self.qkv = scope.put(np.zeros((rows, self.row), dtype))
        self.shared = c.put(scope)
        e = np.dtype(dtype).itemsize
        part = lambda at: cache_test.Slice(self.qkv, at * dim * e, (rows * self.row - at * dim) * e, dtype)
        self.frequencies = (100.0 ** (-np.arange(dim // 2) / (dim // 2))).astype(np.float32)
        self.rotated, self.attended = (scope.put(np.zeros((rows, heads * dim), dtype)) for _ in range(2))
        self.head = q4.make(rng, dtype, rows, heads * dim, columns, 64, bias=True)
        self.head["scales"] = self.head["scales"] * dtype(4)
        self.logits = scope.put(np.zeros((rows, columns), dtype))
        self.case = verify.make(rng, dtype, counts, columns, stride=columns)
        self.verify_buffers = {n: scope.put(self.case[n]) for n in ("draft", "tokens", "uniforms", "draws")}
        self.accepted, self.next = (scope.put(np.zeros(len(counts), np.uint32)) for _ in range(2))
        self.ops = [
            abi.CacheAppendOp(ctx, queries=part(0), query_stride=self.row, query_output=self.rotated, keys=part(heads),
                              key_stride=self.row, values=part(heads + kv_heads), value_stride=self.row, heads=heads,
                              rotary_dim=dim, frequencies=scope.put(self.frequencies), **self.shared),
            abi.CacheAttentionOp(ctx, queries=self.rotated, output=self.attended, heads=heads, window=window, **self.shared),
            abi.Q4GemmOp(ctx, a=self.attended, packed=scope.put(abi.pack_q4(self.head["codes"])),
                         scales=scope.put(self.head["scales"]), bias=scope.put(self.head["bias"]), output=self.logits,
                         rows=rows, inner=heads * dim, columns=columns, group_size=64),
            abi.DraftVerifyOp(ctx, target=self.logits, rows=rows, sequences=len(counts), columns=columns,
                              row_starts=self.shared["row_starts"], accepted=self.accepted, next_tokens=self.next,
                              **self.verify_buffers)]

    def feed(self, grow=True):
        """New rows, and lengths that count them."""
        c = self.cache
        if grow:
            c.lengths = (c.lengths + np.array(c.counts)).astype(np.uint32)
        self.new = self.rng.standard_normal((c.rows, self.row)).astype(self.dtype)
        self.qkv.upload(self.new)
        c.device["lengths"].upload(c.lengths)
        self.case["uniforms"] = self.rng.random(c.rows).astype(np.float32)
        self.verify_buffers["uniforms"].upload(self.case["uniforms"])
        self.ctx.synchronize()

    def enqueue(self, stream=None):
        for op in self.ops:
            op.enqueue(0, stream)

    def check(self):
        c, dim, kv, heads = self.cache, self.cache.dim, self.cache.kv_heads, self.heads
        got = [self.rotated.download(), c.device["key_cache"].download(), c.device["value_cache"].download()]
        cut = [self.new[:, :heads * dim], self.new[:, heads * dim:(heads + kv) * dim], self.new[:, (heads + kv) * dim:]]
        cache_test.check_append(c, got, *cut, self.frequencies, "halves", heads=heads)
        c.keys, c.values = got[1], got[2]
        attended = self.attended.download()
        cache_test.check_attention(c, attended, got[0], heads, window=self.window)
        logits = self.logits.download()
        q4.check(logits, dict(self.head, a=attended))
        margins, case = [], self.case
        want = verify.formula(logits, case["draft"], case["tokens"], case["starts"], case["uniforms"], case["draws"], 1.0,
                              False, margins)
        assert min(margins) > verify.MARGIN
        np.testing.assert_array_equal(self.accepted.download(), want[0])
        np.testing.assert_array_equal(self.next.download(), want[1])

    def release(self):
        for op in self.ops:
            op.release()


SHAPES = pytest.mark.parametrize("counts,lengths", [([1], [5]), ([4, 1, 6], [20, 3, 100]), ([60, 3, 40], [0, 200, 17])])


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@SHAPES
def test_steps(abi, ctx, scope, dtype, counts, lengths):
    step = Decoder(abi, ctx, scope, np.random.default_rng(1), dtype, counts, lengths)
    for _ in range(4):
        step.feed()
        step.enqueue()
        ctx.synchronize()
        step.check()
    step.release()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@SHAPES
def test_replayed_steps(abi, ctx, scope, dtype, counts, lengths):
    """One graph for all steps: lengths and rows are read when it runs."""
    step = Decoder(abi, ctx, scope, np.random.default_rng(2), dtype, counts, lengths, window=50)
    graph = abi.Graph.capture(ctx, ctx.stream)
    with graph:
        step.enqueue(ctx.stream)
    for i in range(4):
        step.feed()
        graph.launch()
        ctx.synchronize()
        step.check()
        if i % 2:  # eager work between the replays, of the same step
            step.feed(grow=False)
            step.enqueue()
            ctx.synchronize()
            step.check()
    graph.release()
    step.release()


def test_two_graphs_and_two_streams(abi, ctx, scope):
    """Two decoders, each with its own graph, at once on two streams."""
    rng = np.random.default_rng(3)
    steps = [Decoder(abi, ctx, scope, rng, np.float16, [2, 5], [30, 300]),
             Decoder(abi, ctx, scope, rng, np.float16, [1] * 9, list(range(10, 370, 40)))]
    other = ctypes.c_void_p()
    abi.check(abi.load().pk_stream_create(ctx.handle, ctypes.byref(other)))
    streams, graphs = [ctx.stream, other], []
    for step, stream in zip(steps, streams):
        graphs.append(abi.Graph.capture(ctx, stream))
        with graphs[-1]:
            step.enqueue(stream)
    for _ in range(3):
        for step in steps:
            step.feed()
        for _ in range(5):  # the same step again gives the same
            for graph, stream in zip(graphs, streams):
                graph.launch(stream)
        ctx.synchronize(other)
        ctx.synchronize()
        for step in steps:
            step.check()
    for graph in graphs:
        graph.release()
    for step in steps:
        step.release()
    abi.check(abi.load().pk_stream_destroy(ctx.handle, other))


def test_in_order_on_the_default_stream(abi, ctx, scope):
    """hipStreamLegacy by its handle: behind the copies before, in front of those after."""
    step = Decoder(abi, ctx, scope, np.random.default_rng(4), np.float16, [3, 1], [40, 10])
    step.feed()
    step.enqueue()
    ctx.synchronize()
    step.check()
    want = [x.download() for x in (step.attended, step.logits, step.next)]
    rows = scope.put(step.new)
    long = [scope.empty(1 << 28, np.uint8) for _ in range(2)]
    zeros = scope.put(np.zeros_like(step.new))
    for _ in range(3):
        ctx.copy(step.qkv, zeros, 1)
        step.enqueue(1)
        for i in range(3):
            ctx.copy(long[i % 2], long[1 - i % 2], 1)
        ctx.copy(step.qkv, rows, 1)
        step.enqueue(1)
        kept = [scope.empty(x.shape, x.dtype) for x in want]
        for to, x in zip(kept, (step.attended, step.logits, step.next)):
            ctx.copy(to, x, 1)
        ctx.copy(step.qkv, zeros, 1)
        ctx.synchronize(1)
        for got, x in zip(kept, want):
            np.testing.assert_array_equal(got.download(), x)
    step.release()


def test_results_do_not_change_from_run_to_run(abi, ctx, scope):
    """Parts of long sequences are joined in a fixed order."""
    step = Decoder(abi, ctx, scope, np.random.default_rng(5), np.float16, [1, 1, 7], [100, 5000, 3000], most=6000)
    step.feed()
    first = None
    for _ in range(20):
        step.enqueue()
        ctx.synchronize()
        got = step.attended.download()
        first = got if first is None else first
        np.testing.assert_array_equal(got.view(np.uint16), first.view(np.uint16))
    step.release()


def test_ops_outlive_their_context(abi, scope):
    own = abi.Context(0)
    inner = Scope(own)
    step = Decoder(abi, own, inner, np.random.default_rng(6), np.float16, [2, 1], [20, 700], most=800)
    step.feed()
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


def test_more_sequences_than_the_capacity(abi, ctx, scope):
    step = Decoder(abi, ctx, scope, np.random.default_rng(7), np.float16, [2, 1], [20, 70])
    for op in (step.ops[0], step.ops[1], step.ops[3]):
        with pytest.raises(abi.PaletteRangeError, match=r"active sequences must be in \[1, 2\]"):
            op.enqueue(3)
    step.release()


def test_events(abi, ctx, scope):
    step = Decoder(abi, ctx, scope, np.random.default_rng(8), np.float16, [2, 1], [20, 900], most=1000)
    step.feed()
    start, end = abi.Event(ctx), abi.Event(ctx)
    for op in step.ops:
        op.enqueue(start=start, end=end)
        ctx.synchronize()
        assert 0 < start.elapsed_ms(end) < 100
    step.check()
    step.release()
