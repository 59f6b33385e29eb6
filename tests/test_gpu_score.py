"""Token scores (pk_score) against float64.

Tolerances: a difference to the maximum and its product with 1 / T are off by
two f32 half steps of themselves, exp by two more and its argument's, a sum of
V terms over at least 64 lanes by V / 64 + 32 half steps. With r the sum of the
others relative to the maximum, log1p(r) moves by that times r / (1 + r), and
the entropy's second term by that times itself. Alternatives are exact."""
import numpy as np
import pytest

from test_gpu_parity import Scope

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -24
NONE = 0xFFFFFFFF


@pytest.fixture
def scope(ctx):
    s = Scope(ctx)
    yield s
    s.close()


def make(rng, dtype, rows, columns, *, peak=True, masked=0.0, std=2.5):
    x = rng.standard_normal((rows, columns)) * std
    if peak:
        x[np.arange(rows), rng.integers(0, columns, rows)] += rng.uniform(0, 14, rows)
    if masked:
        x[rng.random((rows, columns)) < masked] = -np.inf
    return x.astype(dtype), rng.integers(0, columns, rows).astype(np.uint32)


def reference(logits, tokens, k, temperature=1.0):
    """log probs, entropies, top tokens, top log probs, and the tolerances of
    the three floats; rows as pk_score.h says."""
    inverse = np.float64(np.float32(1.0) / np.float32(temperature))
    rows, columns = logits.shape
    z = logits.astype(np.float64) * inverse
    with np.errstate(invalid="ignore", divide="ignore"):
        m = np.max(z, 1, keepdims=True)
        d = z - m
        e = np.exp(d)
        first = np.argmax(z, 1)
        rest = e.copy()
        rest[np.arange(rows), first] = 0
        r = rest.sum(1)
        t = -np.where(e > 0, e * d, 0).sum(1)
        bad = ~np.isfinite(r) | np.isnan(z).any(1) | np.isposinf(z).any(1)
        empty = (logits == -np.inf).all(1)
        bad &= ~empty
        log_p = d - np.log1p(r)[:, None]
        entropy = np.log1p(r) + t / (1 + r)
    relative = (columns / 64 + 64) * STEP
    share = np.where(empty | bad, 0, r / (1 + r))
    spread = relative * share + 4 * STEP * np.where(empty | bad, 0, np.log1p(np.where(empty | bad, 0, r)))
    log_p[bad], entropy[bad] = np.nan, np.nan
    log_p[empty], entropy[empty] = -np.inf, 0.0
    with np.errstate(invalid="ignore"):
        tol_p = spread[:, None] + 4 * STEP * np.where(np.isfinite(d), np.abs(d), 0) + 1e-37
    tol_h = spread + np.where(empty | bad, 0, relative * np.abs(np.where(empty | bad, 0, t)) / (1 + np.where(empty | bad, 0, r))) + 1e-37
    known = tokens < columns
    at = np.where(known, tokens, 0).astype(np.int64)
    given, given_tol = log_p[np.arange(rows), at], tol_p[np.arange(rows), at]
    given[~known] = np.nan
    given[tokens == NONE] = 0.0
    raw = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    order = np.argsort(-raw, axis=1, kind="stable")[:, :k]
    if order.shape[1] < k:
        order = np.concatenate([order, np.zeros((rows, k - order.shape[1]), order.dtype)], 1)
        beyond = np.arange(k)[None, :] >= columns
    else:
        beyond = np.zeros((1, k), bool)
    none = beyond | (np.take_along_axis(raw, order, 1) == -np.inf)
    top = np.where(none, NONE, order).astype(np.uint32)
    top_p = np.where(none, -np.inf, np.take_along_axis(log_p, order, 1))
    return given, entropy, top, top_p, given_tol, tol_h, np.take_along_axis(tol_p, order, 1)


def run(abi, ctx, scope, logits, tokens, k, *, temperature=None, stride=0, lead=0, active=0, op_of=None):
    rows, columns = logits.shape
    stride = stride or columns
    whole = np.full(lead + rows * stride, 99, logits.dtype)  # what lies between the rows would win
    whole[lead:].reshape(rows, stride)[:, :columns] = logits
    buffer = scope.put(whole)

    class View:
        ptr = buffer.ptr + lead * logits.dtype.itemsize
        nbytes = ((rows - 1) * stride + columns) * logits.dtype.itemsize
        dtype = logits.dtype
    outs = dict(log_probs=scope.put(np.full(rows, 5, np.float32)), entropies=scope.put(np.full(rows, 5, np.float32)))
    if k:
        outs.update(top_tokens=scope.put(np.full((rows, k), 5, np.uint32)),
                    top_log_probs=scope.put(np.full((rows, k), 5, np.float32)))
    op = abi.TokenScoreOp(ctx, logits=View, rows=rows, columns=columns, row_stride=stride, tokens=scope.put(tokens),
                          alternatives=k, temperature=temperature, **outs)
    try:
        op.enqueue(active)
        ctx.synchronize()
    finally:
        op.release()
    got = [outs[n].download() for n in ("log_probs", "entropies")]
    return got + ([outs[n].download() for n in ("top_tokens", "top_log_probs")] if k else [])


def near(got, want, tol, what):
    got = got.astype(np.float64)
    # beyond the largest f32, as the lowest logit below the highest one
    # (-2 * 3.4e38), a value rounds to infinity
    want = np.where(np.abs(want) > np.finfo(np.float32).max, np.copysign(np.inf, want), want)
    plain = np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want), err_msg=what)
    np.testing.assert_array_equal(got[~plain & ~np.isnan(want)], want[~plain & ~np.isnan(want)], err_msg=what)
    far = np.abs(got[plain] - want[plain]) - tol[plain] - STEP * np.abs(want[plain])
    assert (far <= 0).all(), (what, far.max())


def check(got, logits, tokens, k, temperature=1.0, rows=None):
    n = rows or len(logits)
    lp, h, top, top_p, tol_lp, tol_h, tol_top = reference(logits[:n], tokens[:n], k, temperature)
    near(got[0][:n], lp, tol_lp, "log_probs")
    near(got[1][:n], h, tol_h, "entropies")
    if k:
        np.testing.assert_array_equal(got[2][:n], top)
        near(got[3][:n], top_p, tol_top, "top_log_probs")


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,columns", [(1, 1), (2, 2), (3, 5), (5, 63), (4, 64), (3, 65), (7, 511), (6, 1025),
                                          (300, 1025), (2, 4096), (3, 5001), (2, 16384), (2, 32000), (5, 50257),
                                          (1, 131072), (9, 70001), (2, 262144), (520, 2000),
                                          (300, 16001), (90, 66000)])
def test_matches_float64(abi, ctx, scope, dtype, rows, columns):
    rng = np.random.default_rng(rows * 11 + columns)
    logits, tokens = make(rng, dtype, rows, columns)
    for k in (4, 0, 32):
        check(run(abi, ctx, scope, logits, tokens, k), logits, tokens, k)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("columns", [5, 1025, 3001, 40000])
@pytest.mark.parametrize("stride,lead", [(0, 1), (3, 0), (7, 5), (8, 8)])
def test_strides_and_alignment(abi, ctx, scope, dtype, columns, stride, lead):
    """Rows from any element on; between them lie larger logits."""
    logits, tokens = make(np.random.default_rng(columns), dtype, 5, columns)
    got = run(abi, ctx, scope, logits, tokens, 8, stride=columns + stride, lead=lead)
    check(got, logits, tokens, 8)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("temperature", [0.01, 0.7, 1.5, 1000.0])
@pytest.mark.parametrize("columns", [1025, 33000])
def test_temperature(abi, ctx, scope, dtype, temperature, columns):
    logits, tokens = make(np.random.default_rng(3), dtype, 4, columns)
    check(run(abi, ctx, scope, logits, tokens, 5, temperature=temperature), logits, tokens, 5, temperature)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("columns", [7, 300, 1025, 20000, 140001])
def test_masks(abi, ctx, scope, dtype, columns):
    """Masks of minus infinity and of the type's lowest value, rows with one
    token left, with none, and with fewer than alternatives."""
    rng = np.random.default_rng(columns)
    logits, tokens = make(rng, dtype, 9, columns, masked=0.3)
    logits[1] = -np.inf
    logits[2] = -np.inf
    logits[2, columns // 2] = -3.0
    logits[3, 2:] = -np.inf
    logits[4] = np.finfo(dtype).min
    logits[5, : columns // 2] = np.finfo(dtype).min
    logits[6] = np.finfo(dtype).min
    logits[6, -1] = np.finfo(dtype).max
    tokens[2], tokens[6] = columns // 2, columns - 1
    check(run(abi, ctx, scope, logits, tokens, 6), logits, tokens, 6)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("columns", [40, 1025, 9000, 140001])
def test_ties_go_to_the_lowest_index(abi, ctx, scope, dtype, columns):
    """All equal, a few values, zeros of both signs, rising and falling rows."""
    rng = np.random.default_rng(columns)
    logits, tokens = make(rng, dtype, 7, columns)
    logits[0] = 1.5
    logits[1] = rng.integers(-2, 3, columns)
    logits[2] = np.where(rng.random(columns) < 0.5, 0.0, -0.0)
    logits[3] = np.arange(columns) / columns * 8
    logits[4] = -logits[3]
    logits[5] = np.repeat(rng.standard_normal(-(-columns // 32)), 32)[:columns]
    for k in (1, 9, 32):
        check(run(abi, ctx, scope, logits, tokens, k), logits, tokens, k)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("columns", [65, 1025, 90000])
def test_infinities_and_nan(abi, ctx, scope, dtype, columns):
    """NaN and plus infinity stay in their rows, and their alternatives are
    ordered without the NaNs."""
    logits, tokens = make(np.random.default_rng(5), dtype, 8, columns)
    logits[1, 3], logits[2, 7], logits[4] = np.nan, np.inf, np.nan
    logits[5] = -np.inf
    logits[5, 1] = np.nan
    logits[6, 60:62] = np.inf
    tokens[1] = NONE
    check(run(abi, ctx, scope, logits, tokens, 4), logits, tokens, 4)


@pytest.mark.parametrize("dtype,bits,signalling", [(np.float16, np.uint16, 0x7D00), (np.float32, np.uint32, 0x7FA00000)])
@pytest.mark.parametrize("columns", [300, 9000])
def test_signalling_nan(abi, ctx, scope, dtype, bits, signalling, columns):
    """A NaN that arithmetic would turn quiet hides none of its neighbours."""
    logits, tokens = make(np.random.default_rng(columns), dtype, 4, columns)
    for row in range(3):
        at = int(np.argmax(logits[row])) ^ (row + 1)  # beside the largest, in its vector
        logits.view(bits)[row, min(at, columns - 1)] = signalling
    got = run(abi, ctx, scope, logits, tokens, 4)
    check(got, logits, tokens, 4)


@pytest.mark.parametrize("dtype,bits,signalling", [(np.float16, np.uint16, 0x7D00), (np.float32, np.uint32, 0x7FA00000)])
@pytest.mark.parametrize("columns", [31, 300, 1900, 9000])
def test_signalling_nan_outside_the_vectors(abi, ctx, scope, dtype, bits, signalling, columns):
    """The element before the first 16-byte boundary, and the one of a lane
    behind the last, beside the largest logit in the same lane's vector."""
    lead = 16 // np.dtype(dtype).itemsize - 1
    logits, tokens = make(np.random.default_rng(columns), dtype, 2, columns, peak=False)
    stride = columns + -columns % (lead + 1)
    logits.view(bits)[:, 0] = signalling
    logits[0, 1], logits[1, 2] = 60, 60
    check(run(abi, ctx, scope, logits, tokens, 4, lead=lead, stride=stride), logits, tokens, 4)
    logits[:, 0] = 1
    logits.view(bits)[:, -1] = signalling
    check(run(abi, ctx, scope, logits, tokens, 4, stride=stride), logits, tokens, 4)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("temperature", [2.0 ** -20, 2.0 ** 20])
def test_temperature_limits(abi, ctx, scope, dtype, temperature):
    logits, tokens = make(np.random.default_rng(4), dtype, 3, 2000)
    check(run(abi, ctx, scope, logits, tokens, 3, temperature=temperature), logits, tokens, 3, temperature)


@pytest.mark.parametrize("temperature", [2.0 ** -20, 2.0 ** -16])
def test_large_f16_logits_at_low_temperatures(abi, ctx, scope, temperature):
    """Where the product of the largest logit and 1 / T passes 2^31, its
    rounding alone is worth an exponent that f32 does not hold."""
    logits, tokens = make(np.random.default_rng(6), np.float16, 64, 300)
    logits[:32] = -np.abs(logits[:32]) - 2000
    logits[np.arange(64), tokens] = np.linspace(-1500, -200, 64)
    logits[32:, 7] = np.linspace(2000, 65504, 32)
    logits[40:, 9] = logits[40:, 7]
    check(run(abi, ctx, scope, logits, tokens, 4, temperature=temperature), logits, tokens, 4, temperature)


def test_tokens_outside(abi, ctx, scope):
    logits, tokens = make(np.random.default_rng(5), np.float16, 6, 1025)
    tokens[1], tokens[2], tokens[3], tokens[4] = NONE, 1025, 1031, NONE - 1
    got = run(abi, ctx, scope, logits, tokens, 2, stride=1032)
    check(got, logits, tokens, 2)
    assert got[0][1] == 0 and np.isnan(got[0][2:5]).all()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("columns", [1025, 40000])
def test_certain_rows_keep_their_digits(abi, ctx, scope, dtype, columns):
    """Log probabilities near zero and entropies far below an f32 step of one."""
    logits, tokens = make(np.random.default_rng(6), dtype, 5, columns, peak=False, std=1.0)
    for row, height in enumerate((25, 35, 50, 80, 12)):
        logits[row, 17] = height
    tokens[:] = 17
    got = run(abi, ctx, scope, logits, tokens, 2)
    check(got, logits, tokens, 2)
    assert (got[0] < 0).all() and (got[1] > 0).all()


@pytest.mark.parametrize("columns", [300, 60000])
def test_active_rows_leave_the_others(abi, ctx, scope, columns):
    logits, tokens = make(np.random.default_rng(8), np.float16, 12, columns)
    got = run(abi, ctx, scope, logits, tokens, 3, active=7)
    check(got, logits, tokens, 3, rows=7)
    assert all((g[7:] == 5).all() for g in got)


def test_single_outputs(abi, ctx, scope):
    """Each output on its own."""
    logits, tokens = make(np.random.default_rng(9), np.float16, 4, 2000)
    lp, h, top, top_p, tol_lp, tol_h, tol_top = reference(logits, tokens, 3)
    x, t = scope.put(logits), scope.put(tokens)
    out = scope.empty(4, np.float32)
    ids, probs = scope.empty((4, 3), np.uint32), scope.empty((4, 3), np.float32)
    for kw, result, want, tol in ((dict(tokens=t, log_probs=out), out, lp, tol_lp), (dict(entropies=out), out, h, tol_h),
                                  (dict(alternatives=3, top_tokens=ids, top_log_probs=probs), probs, top_p, tol_top)):
        op = abi.TokenScoreOp(ctx, logits=x, rows=4, columns=2000, **kw)
        op.enqueue()
        ctx.synchronize()
        op.release()
        near(result.download(), want, tol, "single")
    np.testing.assert_array_equal(ids.download(), top)


@pytest.mark.parametrize("rows,columns", [(30, 1025), (3, 131072)])
def test_graph(abi, ctx, scope, rows, columns):
    rng = np.random.default_rng(10)
    logits, tokens = make(rng, np.float16, rows, columns)
    x = scope.put(logits)
    outs = dict(log_probs=scope.empty(rows, np.float32), entropies=scope.empty(rows, np.float32),
                top_tokens=scope.empty((rows, 8), np.uint32), top_log_probs=scope.empty((rows, 8), np.float32))
    op = abi.TokenScoreOp(ctx, logits=x, rows=rows, columns=columns, tokens=scope.put(tokens), alternatives=8, **outs)
    graph = abi.Graph.capture(ctx, ctx.stream)
    with graph:
        op.enqueue(0, ctx.stream)
    for _ in range(3):
        logits, _ = make(rng, np.float16, rows, columns)
        x.upload(logits)
        graph.launch()
        ctx.synchronize()
        check([o.download() for o in outs.values()], logits, tokens, 8)
        op.enqueue(1)
        ctx.synchronize()
    graph.release()
    op.release()
