"""The norms around a block (pk_block_norm) against float64.

Tolerances: the kernel computes in f32 and rounds an output once, by at most
half a step of its type (eps / 2 of the value). A mean of C values is off by
at most 64 f32 half steps of the mean magnitude (a lane sums up to 32 values,
the wavefront's and the workgroup's sums add 10), a variance by as many of
itself, so every term of the sums below is off by at most 128 half steps of
its magnitude, and what the first output is off by reaches the second divided
by its deviation."""
import numpy as np
import pytest

from test_gpu_parity import Scope

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -24


@pytest.fixture
def scope(ctx):
    s = Scope(ctx)
    yield s
    s.close()


def norm64(x, kind, gamma, beta, epsilon, off):
    """(norm(x), how far f32 may be from it) where x is already off by `off`."""
    mean = x.mean(-1, keepdims=True) if kind == "layer" else 0.0
    sigma = np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + epsilon)
    size = np.abs(x) + np.abs(x).mean(-1, keepdims=True)
    g, b = gamma.astype(np.float64), 0.0 if beta is None else beta.astype(np.float64)
    y = (x - mean) / sigma * g + b
    # an error of x moves the mean and the deviation too: at most three times itself in units of sigma
    spread = np.abs(off) + np.abs(off).max(-1, keepdims=True) * (1 + np.abs(x - mean) / sigma)
    return y, (128 * STEP * size + 2 * spread) / sigma * np.abs(g) + 128 * STEP * np.abs(b)


def reference(case):
    """[(output, tolerance)] in float64, for y and the norm of it."""
    x = case["input"].astype(np.float64)
    off = np.zeros_like(x)
    kind, epsilon = case["kind"], case.get("epsilon") or (0.0 if case.get("epsilon") == 0 else 1e-5)
    if case.get("gamma") is not None:
        x, off = norm64(x, kind, case["gamma"], case.get("beta"), epsilon, off)
    scale = case.get("residual_scale")
    scale = 1.0 if scale is None else np.float64(np.float32(scale))
    factor = np.full_like(x, scale)
    if case.get("gate") is not None:
        each = case.get("gate_rows", 1)
        at = np.arange(len(x)) // each if each else np.zeros(len(x), int)
        factor = factor * case["gate"].astype(np.float64)[at]
    off = np.abs(factor) * off + 8 * STEP * np.abs(factor * x)
    y = factor * x
    if case.get("residual") is not None:
        y = y + case["residual"].astype(np.float64)
        off = off + 2 * STEP * np.abs(y)
    half = np.finfo(case["input"].dtype).eps / 2
    tiny = np.finfo(case["input"].dtype).smallest_subnormal
    outs = [(y, half * np.abs(y) + 2 * off + tiny)]
    if case.get("next_gamma") is not None:
        z, off = norm64(y, kind, case["next_gamma"], case.get("next_beta"), epsilon, off)
        outs.append((z, half * np.abs(z) + 2 * off + tiny))
    return outs


def strided(scope, host, stride, lead):
    """The rows of `host` in a buffer of rows of `stride`, `lead` elements in:
    (buffer, view with the pointer of the first element, stride)."""
    rows, channels = host.shape
    whole = np.full(lead + rows * stride + 8, 77, host.dtype)
    whole[lead:lead + rows * stride].reshape(rows, stride)[:, :channels] = host
    buffer = scope.put(whole)

    class View:
        ptr = buffer.ptr + lead * host.dtype.itemsize
        nbytes = ((rows - 1) * stride + channels) * host.dtype.itemsize
        dtype = host.dtype

        @staticmethod
        def download():
            got = buffer.download()
            body = got[lead:lead + rows * stride].reshape(rows, stride)
            assert (got[:lead] == 77).all() and (body[:, channels:] == 77).all() and (got[lead + rows * stride:] == 77).all()
            return body[:, :channels]
    return View


def make(rng, dtype, rows, channels, kind="layer", gate="none", post=True, next=True, residual=True, beta=True,
         offset=0.3, **more):
    def values(n, mean=0.0, std=1.0):
        return (rng.standard_normal((n, channels)) * std + mean).astype(dtype)

    def vector(mean):
        return (rng.standard_normal(channels) * 0.2 + mean).astype(np.float32)
    case = dict(kind=kind, input=values(rows, offset, 1.5), **more)
    if post:
        case["gamma"], case["beta"] = vector(1.0), vector(0.0) if beta else None
    if gate != "none":
        each = {"row": 1, "all": 0}.get(gate, gate)
        case["gate"], case["gate_rows"] = values(-(-rows // each) if each else 1), each
    if residual:
        case["residual"] = values(rows, 0.1, 2.0)
        case.setdefault("residual_scale", 0.5)
    if next:
        case["next_gamma"], case["next_beta"] = vector(1.0), vector(0.0) if beta else None
    return case


def run(abi, ctx, scope, case, *, active=0, stride=0, lead=0, stream=None, out_on=None, next_on=None):
    rows, channels = case["input"].shape

    def put(a):
        if stride:
            return strided(scope, a, stride, lead)
        return scope.put(a)
    kw = {n: put(case[n]) for n in ("input", "gate", "residual") if case.get(n) is not None}
    kw.update({n: scope.put(case[n]) for n in ("gamma", "beta", "next_gamma", "next_beta") if case.get(n) is not None})
    kw.update({n: case[n] for n in ("kind", "gate_rows", "residual_scale", "epsilon") if n in case})
    fill = np.full((rows, channels), 321, case["input"].dtype)
    kw["output"] = kw[out_on] if out_on else put(fill)
    if "next_gamma" in kw:
        kw["next_output"] = kw[next_on] if next_on else put(fill)
    if stride:
        kw.update({n + "_stride": stride for n in ("input", "gate", "residual", "output", "next_output") if n in kw})
    op = abi.BlockNormOp(ctx, rows=rows, channels=channels, **kw)
    try:
        op.enqueue(active, stream)
        ctx.synchronize(stream)
    finally:
        op.release()
    return [kw[n].download() for n in ("output", "next_output") if n in kw]


def check(got, case, rows=None):
    for g, (want, tol) in zip(got, reference(case), strict=True):
        n = rows or len(want)
        far = np.abs(g[:n].astype(np.float64) - want[:n]) - tol[:n]
        assert (far <= 0).all(), (far.max(), np.unravel_index(far.argmax(), far.shape))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,channels", [(1, 1), (3, 5), (7, 64), (5, 640), (2, 1000), (9, 1024), (4, 1025), (3, 2048),
                                           (2, 2056), (2, 4096), (3, 4097), (2, 8192), (2, 8200), (1, 16383),
                                           (2, 16384), (1503, 128)])
def test_matches_float64(abi, ctx, scope, dtype, rows, channels):
    rng = np.random.default_rng(rows * 100003 + channels)
    for kind, gate in (("layer", "none"), ("rms", "row")):
        case = make(rng, dtype, rows, channels, kind, gate)
        check(run(abi, ctx, scope, case), case)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("gate", ["none", "row", "all", 3, 100])
@pytest.mark.parametrize("post,next,residual,beta", [(True, True, True, True), (False, True, True, False),
                                                     (True, False, False, True), (False, False, True, True),
                                                     (True, True, False, False)])
def test_parts(abi, ctx, scope, dtype, kind, gate, post, next, residual, beta):
    case = make(np.random.default_rng(5), dtype, 10, 264, kind, gate, post, next, residual, beta)
    check(run(abi, ctx, scope, case), case)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("channels,stride,lead", [(640, 640, 8), (640, 648, 0), (640, 641, 0), (640, 640, 1), (7, 9, 3),
                                                  (2100, 4200, 0)])
def test_strides_and_alignment(abi, ctx, scope, dtype, channels, stride, lead):
    """Rows inside wider ones, and starts that are not on 16 bytes; what lies
    between the rows stays."""
    case = make(np.random.default_rng(channels + stride), dtype, 6, channels, "rms", "row")
    check(run(abi, ctx, scope, case, stride=stride, lead=lead), case)


@pytest.mark.parametrize("out_on,next_on", [("input", None), ("residual", None), (None, "residual"),
                                            ("residual", "input")])
def test_outputs_on_the_inputs(abi, ctx, scope, out_on, next_on):
    for channels in (640, 3000, 9001):
        case = make(np.random.default_rng(channels), np.float16, 9, channels, gate="all")
        check(run(abi, ctx, scope, case, out_on=out_on, next_on=next_on), case)


def test_columns_of_one_buffer(abi, ctx, scope):
    """Value and gate as the halves of one product's rows."""
    rng = np.random.default_rng(8)
    case = make(rng, np.float16, 11, 320, gate="row")
    both = scope.put(np.concatenate([case["input"], case["gate"]], axis=1))

    class Half:
        dtype = np.dtype(np.float16)

        def __init__(self, at):
            self.ptr, self.nbytes = both.ptr + at * 640, (10 * 640 + 320) * 2
    out, nxt = scope.empty((11, 320), np.float16), scope.empty((11, 320), np.float16)
    put = {n: scope.put(case[n]) for n in ("gamma", "beta", "residual", "next_gamma", "next_beta")}
    op = abi.BlockNormOp(ctx, rows=11, channels=320, input=Half(0), input_stride=640, gate=Half(1), gate_stride=640,
                         output=out, next_output=nxt, residual_scale=0.5, **put)
    op.enqueue()
    ctx.synchronize()
    op.release()
    check([out.download(), nxt.download()], case)


def test_active_rows_leave_the_others(abi, ctx, scope):
    case = make(np.random.default_rng(3), np.float16, 40, 1024, gate=16)
    got = run(abi, ctx, scope, case, active=25)
    check(got, case, rows=25)
    assert all((g[25:] == 321).all() for g in got)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_hard_rows(abi, ctx, scope, dtype):
    """Constant rows, rows far from zero, rows of zeros, and epsilon 0 and 0.5."""
    rng = np.random.default_rng(11)
    case = make(rng, dtype, 8, 512, offset=0.0)
    x = case["input"]
    x[0], x[1], x[2] = 3.0, 0.0, 1000 + rng.integers(0, 3, 512)
    x[3], x[3, 0] = 0.001 * x[3], 4000.0
    case["residual"][1] = 0.0
    check(run(abi, ctx, scope, case), case)
    for epsilon in (0.5, 0.0):
        case = make(rng, dtype, 4, 300, epsilon=epsilon)
        check(run(abi, ctx, scope, case), case)


@pytest.mark.parametrize("channels", [640, 5000])
def test_infinities_and_nan_stay_in_their_rows(abi, ctx, scope, channels):
    case = make(np.random.default_rng(2), np.float16, 9, channels, gate="row")
    clean = run(abi, ctx, scope, case)
    case["input"][1, 5], case["input"][4, 7], case["residual"][6, 1], case["gate"][8, 0] = np.inf, np.nan, -np.inf, np.nan
    got = run(abi, ctx, scope, case)
    for g, c in zip(got, clean):
        for row in (0, 2, 3, 5, 7):
            np.testing.assert_array_equal(g[row].view(np.uint16), c[row].view(np.uint16))
    assert np.isnan(got[0][1]).all() and np.isnan(got[0][4]).all() and np.isnan(got[1][[1, 4, 6, 8]]).all()
    assert got[0][6, 1] == -np.inf and np.isfinite(np.delete(got[0][6], 1)).all()
    assert np.isnan(got[0][8, 0]) and np.isfinite(got[0][8, 1:]).all()


def test_streams_and_graph(abi, ctx, scope):
    """One op on its context's stream and on another at once, and replayed from
    a graph with changed inputs between the replays."""
    rng = np.random.default_rng(4)
    case = make(rng, np.float16, 33, 1024, gate="all")
    kw = {n: scope.put(case[n]) for n in ("input", "gate", "residual", "gamma", "beta", "next_gamma", "next_beta")}
    out, nxt = scope.empty((33, 1024), np.float16), scope.empty((33, 1024), np.float16)
    op = abi.BlockNormOp(ctx, rows=33, channels=1024, gate_rows=0, residual_scale=0.5, output=out, next_output=nxt, **kw)
    import ctypes
    other = ctypes.c_void_p()
    abi.check(abi.load().pk_stream_create(ctx.handle, ctypes.byref(other)))
    op.enqueue()
    op.enqueue(0, other)
    ctx.synchronize()
    ctx.synchronize(other)
    check([out.download(), nxt.download()], case)
    graph = abi.Graph.capture(ctx, ctx.stream)
    with graph:
        op.enqueue(0, ctx.stream)
    for _ in range(3):
        case["input"] = (rng.standard_normal((33, 1024))).astype(np.float16)
        kw["input"].upload(case["input"])
        graph.launch()
        ctx.synchronize()
        check([out.download(), nxt.download()], case)
    graph.release()
    op.release()
    abi.check(abi.load().pk_stream_destroy(ctx.handle, other))
