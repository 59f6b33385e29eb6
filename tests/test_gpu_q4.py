"""The product with 4-bit group-scaled weights (pk_q4) against float64.

Tolerances: weights are exact multiples of their scales, products of f16 (or
f32) activations with codes are exact to f32, and a sum over K is off by at
most one f32 step of the sum of magnitudes per accumulation step: K / 4 of
them for f32 operands, K / 32 blocks of 32 for f16 ones, and 64 for joining
parts, scaling and the epilogue. SiLU's exponential multiplies its argument's
rounding by the argument. An output is rounded once, by half a step."""
import numpy as np
import pytest

from test_gpu_block_norm import strided
from test_gpu_parity import Scope

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -23


@pytest.fixture
def scope(ctx):
    s = Scope(ctx)
    yield s
    s.close()


def make(rng, dtype, rows, inner, columns, group, offsets=False, bias=False, activation="none", residual=False,
         residual_scale=None):
    groups = -(-inner // (group or inner))
    case = dict(a=rng.standard_normal((rows, inner)).astype(dtype),
                codes=rng.integers(0, 16, (inner, columns)).astype(np.uint8),
                scales=rng.uniform(0.002, 0.008, (groups, columns)).astype(dtype), group_size=group,
                activation=activation, residual_scale=residual_scale)
    if offsets:
        case["offsets"] = (rng.standard_normal((groups, columns)) * 0.004).astype(dtype)
    if bias:
        case["bias"] = (rng.standard_normal(columns) * 0.1).astype(np.float32)
    if residual:
        case["residual"] = rng.standard_normal((rows, columns)).astype(dtype)
    return case


def reference(case):
    a, dtype = case["a"].astype(np.float64), case["a"].dtype
    inner, columns = case["codes"].shape
    at = np.arange(inner) // (case["group_size"] or inner)
    scale = case["scales"].astype(np.float64)[at]
    w, size = scale * (case["codes"].astype(np.float64) - 8), np.abs(scale) * 8
    if "offsets" in case:
        offset = case["offsets"].astype(np.float64)[at]
        w, size = w + offset, size + np.abs(offset)
    v = a @ w
    # a sum that later steps add to is off by a step of what is there by then
    magnitude = np.abs(a) @ size
    tol = (inner / (32 if dtype == np.float16 else 4) + 64) * STEP * magnitude
    if "bias" in case:
        v = v + case["bias"].astype(np.float64)
        tol = tol + STEP * np.abs(v)
    if case["activation"] == "silu":
        with np.errstate(over="ignore"):
            y = v / (1 + np.exp(-v))
        tol = 1.1 * tol + (np.abs(v) + 4) * STEP * np.abs(y)
        v = y
    elif case["activation"] == "relu":
        v = np.maximum(v, 0)
    if "residual" in case:
        s = 1.0 if case["residual_scale"] is None else case["residual_scale"]
        v = case["residual"].astype(np.float64) + s * v
        tol = abs(s) * tol + STEP * np.abs(v)
    half = np.finfo(dtype).eps / 2
    return v, half * np.abs(v) + (1 + half) * tol + np.finfo(dtype).smallest_subnormal


def operands(abi, scope, case, strides=None, leads=None):
    strides, leads = strides or {}, leads or {}
    kw = dict(packed=scope.put(abi.pack_q4(case["codes"])), scales=scope.put(case["scales"]))
    for n in ("offsets", "bias"):
        if n in case:
            kw[n] = scope.put(case[n])
    rows, columns = len(case["a"]), case["codes"].shape[1]
    values = {"a": case["a"], "output": np.full((rows, columns), 321, case["a"].dtype),
              "residual": case.get("residual")}
    for n, v in values.items():
        if v is None:
            continue
        if n in strides:
            kw[n], kw[n + "_stride"] = strided(scope, v, strides[n], leads.get(n, 0)), strides[n]
        else:
            kw[n] = scope.put(v)
    return dict(kw, rows=rows, inner=case["a"].shape[1], columns=columns, group_size=case["group_size"],
                activation=case["activation"], residual_scale=case["residual_scale"])


def run(abi, ctx, scope, case, *, active=0, **more):
    kw = operands(abi, scope, case, **more)
    op = abi.Q4GemmOp(ctx, **kw)
    try:
        op.enqueue(active)
        ctx.synchronize()
        return kw["output"].download()
    finally:
        op.release()


def check(got, case, rows=None):
    want, tol = reference(case)
    n = rows or len(want)
    far = np.abs(got[:n].astype(np.float64) - want[:n]) - tol[:n]
    assert (far <= 0).all(), (far.max(), np.unravel_index(far.argmax(), far.shape))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("group", [32, 64, 128, 256, 0])
@pytest.mark.parametrize("rows,inner,columns", [(1, 1, 1), (1, 640, 1032), (3, 33, 17), (2, 100, 40), (16, 256, 16),
                                                (17, 129, 100), (33, 1000, 333), (64, 512, 640), (65, 384, 96),
                                                (130, 320, 200)])
def test_matches_float64(abi, ctx, scope, dtype, group, rows, inner, columns):
    rng = np.random.default_rng(rows * 7 + inner + columns + group)
    for offsets in (False, True):
        case = make(rng, dtype, rows, inner, columns, group, offsets)
        check(run(abi, ctx, scope, case), case)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows", [1, 2, 4, 5, 8, 9, 31, 32, 48, 100, 257])
def test_row_counts(abi, ctx, scope, dtype, rows):
    case = make(np.random.default_rng(rows), dtype, rows, 1024, 520, 128, True, True)
    check(run(abi, ctx, scope, case), case)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("inner,columns", [(4096, 64), (64, 4096), (8192, 16), (2560, 2560), (9000, 129)])
def test_long_axes(abi, ctx, scope, dtype, inner, columns):
    for rows in (1, 20):
        case = make(np.random.default_rng(inner), dtype, rows, inner, columns, 64, bias=True)
        check(run(abi, ctx, scope, case), case)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows", [1, 40, 200])
@pytest.mark.parametrize("activation,bias,residual,scale", [("silu", True, False, None), ("relu", False, True, 0.5),
                                                            ("none", True, True, None), ("silu", False, True, -2.0)])
def test_epilogue(abi, ctx, scope, dtype, rows, activation, bias, residual, scale):
    case = make(np.random.default_rng(6), dtype, rows, 400, 136, 32, False, bias, activation, residual, scale)
    case["scales"] = case["scales"] * dtype(8)  # arguments of SiLU up to some 20
    check(run(abi, ctx, scope, case), case)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows", [3, 20, 150])
def test_strides_and_alignment(abi, ctx, scope, dtype, rows):
    case = make(np.random.default_rng(9), dtype, rows, 200, 72, 64, True, True, "silu", True, 0.5)
    for strides, leads in (({"a": 208}, {}), ({"a": 201, "output": 73}, {"a": 1}), ({"a": 200}, {"a": 3}),
                           ({"residual": 80, "output": 90}, {"output": 5, "residual": 1})):
        check(run(abi, ctx, scope, case, strides=strides, leads=leads), case)


@pytest.mark.parametrize("rows", [1, 30, 150])
def test_every_code_and_its_place(abi, ctx, scope, rows):
    """One-hot rows read single weights back: codes, groups and columns to the bit."""
    rng = np.random.default_rng(1)
    inner, columns = 300, 50
    case = make(rng, np.float32, rows, inner, columns, 64, True)
    picks = rng.permutation(inner)[:rows] if rows <= inner else rng.integers(0, inner, rows)
    case["a"] = np.zeros((rows, inner), np.float32)
    case["a"][np.arange(rows), picks] = 1.0
    scale = case["scales"][np.arange(inner) // 64]
    w = (scale.astype(np.float64) * (case["codes"].astype(np.float64) - 8)).astype(np.float64) + \
        case["offsets"][np.arange(inner) // 64].astype(np.float64)
    got = run(abi, ctx, scope, case).astype(np.float64)
    np.testing.assert_allclose(got, w[picks], rtol=0, atol=2.0 ** -23 * 0.1)


def test_active_rows_leave_the_others(abi, ctx, scope):
    for active in (1, 3, 25, 70):
        case = make(np.random.default_rng(active), np.float16, 90, 256, 96, 128, bias=True)
        got = run(abi, ctx, scope, case, active=active)
        check(got, case, rows=active)
        assert (got[active:] == 321).all()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_infinities_and_nan_stay_in_their_rows(abi, ctx, scope, dtype):
    case = make(np.random.default_rng(2), dtype, 40, 333, 60, 64, True)
    clean = run(abi, ctx, scope, case)
    case["a"][1, 332], case["a"][20, 0] = np.nan, np.inf
    got = run(abi, ctx, scope, case)
    keep = [r for r in range(40) if r not in (1, 20)]
    np.testing.assert_array_equal(got[keep], clean[keep])
    assert np.isnan(got[1]).all() and not np.isfinite(got[20]).any()


@pytest.mark.parametrize("dtype,size", [(np.float16, 2.0 ** -18), (np.float32, 2.0 ** -132)])
@pytest.mark.parametrize("rows", [1, 3, 20, 700])
def test_subnormal_activations(abi, ctx, scope, dtype, size, rows):
    """Activations below the type's smallest normal number keep their value:
    scales bring the outputs back among the normal ones."""
    case = make(np.random.default_rng(rows), dtype, rows, 300, 2064, 64, True)
    case["a"] = (case["a"].astype(np.float64) * size).astype(dtype)
    up = dtype(2.0 ** 10) if dtype == np.float16 else dtype(2.0 ** 60)
    case["scales"], case["offsets"] = case["scales"] * up, case["offsets"] * up
    check(run(abi, ctx, scope, case), case)


@pytest.mark.parametrize("rows", [1, 16, 100])
def test_output_on_the_residual_and_freed_weight(abi, ctx, scope, rows):
    """The output may be the residual; the op keeps its own copy of the weight."""
    case = make(np.random.default_rng(7), np.float16, rows, 256, 128, 32, True, True, "none", True, 0.25)
    kw = operands(abi, scope, case)
    kw["output"] = kw["residual"]
    op = abi.Q4GemmOp(ctx, **kw)
    kw["packed"].upload(np.zeros(kw["packed"].shape, np.uint32))
    kw["scales"].upload(np.zeros(kw["scales"].shape, np.float16))
    kw["offsets"].upload(np.zeros(kw["offsets"].shape, np.float16))
    assert op.weight_bytes() >= 256 * 128 // 2 + 2 * 2 * 8 * 128
    op.enqueue()
    ctx.synchronize()
    check(kw["output"].download(), case)
    op.destroy()
    assert op.weight_bytes() == 0
    with pytest.raises(abi.PaletteDestroyedError):
        op.enqueue()
    op.release()


def test_launches_of_one_count_are_identical(abi, ctx, scope):
    for rows in (1, 8, 70):
        case = make(np.random.default_rng(rows), np.float16, rows, 4096, 512, 64, True)
        first = run(abi, ctx, scope, case)
        np.testing.assert_array_equal(run(abi, ctx, scope, case), first)


def test_graph_and_refused_capture(abi, ctx, scope):
    rng = np.random.default_rng(4)
    case = make(rng, np.float16, 4, 512, 256, 128, bias=True, activation="silu")
    kw = operands(abi, scope, case)
    op = abi.Q4GemmOp(ctx, **kw)
    graph = abi.Graph.capture(ctx, ctx.stream)
    with graph:
        op.enqueue(0, ctx.stream)
        with pytest.raises(abi.PaletteError, match="capturing"):
            abi.Q4GemmOp(ctx, stream=ctx.stream, **kw)
    for _ in range(3):
        case["a"] = rng.standard_normal((4, 512)).astype(np.float16)
        kw["a"].upload(case["a"])
        graph.launch()
        ctx.synchronize()
        check(kw["output"].download(), case)
        op.enqueue(2)  # eager work between the replays
        ctx.synchronize()
    graph.release()
    op.release()


@pytest.mark.parametrize("rows,inner,columns,group,offsets", [
    (250, 300, 1100, 32, True), (87, 300, 5003, 64, True), (60, 1500, 8200, 0, False), (50, 2100, 7000, 128, True),
    (63, 1990, 8190, 32, True), (1000, 2050, 200, 64, False)])
def test_workgroups_of_16_to_64_rows(abi, ctx, scope, rows, inner, columns, group, offsets):
    """Shapes between the few rows of a stream and whole tiles, with edges."""
    case = make(np.random.default_rng(rows), np.float16, rows, inner, columns, group, offsets, bias=True,
                activation="silu", residual=True, residual_scale=0.5)
    strides = dict(output=columns + 1, residual=columns + 3)
    check(run(abi, ctx, scope, case, strides=strides, leads=dict(output=1)), case)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,inner,columns,group", [(640, 300, 2100, 64), (1504, 128, 1032, 0), (1504, 40, 1032, 32),
                                                      (800, 260, 1700, 128)])
def test_tiles(abi, ctx, scope, dtype, rows, inner, columns, group):
    """Many rows and columns: whole tiles, edges in every direction."""
    case = make(np.random.default_rng(inner), dtype, rows, inner, columns, group, inner == 300, bias=True,
                activation="relu", residual=True)
    check(run(abi, ctx, scope, case), case)
    del case["residual"]
    check(run(abi, ctx, scope, case, strides=dict(a=inner + 1, output=columns + 3), leads=dict(a=1, output=1)), case)


@pytest.mark.parametrize("rows,inner,columns,group,offsets", [
    (500, 4200, 512, 128, False), (130, 1100, 5500, 64, True), (49, 8192, 2050, 32, True)])
def test_split_along_k_f32(abi, ctx, scope, rows, inner, columns, group, offsets):
    case = make(np.random.default_rng(rows), np.float32, rows, inner, columns, group, offsets, bias=True,
                activation="silu", residual=True, residual_scale=2.0)
    check(run(abi, ctx, scope, case, strides=dict(a=inner + 1, output=columns + 2)), case)


@pytest.mark.parametrize("rows,inner,columns,group,offsets", [
    (500, 17300, 512, 128, False),  # the last part is one block, K ends in it
    (500, 17408, 512, 0, True), (130, 4100, 5500, 64, True), (40, 8200, 8190, 32, True), (64, 8192, 8192, 128, False)])
def test_split_along_k(abi, ctx, scope, rows, inner, columns, group, offsets):
    """Few tiles of many rows with a long K: parts of K meet in a workspace."""
    rng = np.random.default_rng(rows + inner)
    case = make(rng, np.float16, rows, inner, columns, group, offsets, bias=True, activation="silu", residual=True,
                residual_scale=0.5)
    check(run(abi, ctx, scope, case, strides=dict(a=inner + 3, output=columns + 5, residual=columns + 1),
              leads=dict(output=1)), case)


def test_split_row_counts_launches_and_graph(abi, ctx, scope):
    """One op at row counts with and without parts, launched again and again,
    timed, and replayed from a graph between eager launches."""
    rows, inner, columns = 700, 4200, 4000
    case = make(np.random.default_rng(5), np.float16, rows, inner, columns, 128, True)
    want, tol = reference(case)
    kw = operands(abi, scope, case)
    op = abi.Q4GemmOp(ctx, **kw)
    graph = None
    try:
        def read(n):
            ctx.synchronize()
            got = kw["output"].download()
            far = np.abs(got[:n].astype(np.float64) - want[:n]) - tol[:n]
            assert (far <= 0).all(), (n, far.max())
            assert (got[n:] == 321).all(), n
            return got
        kw["output"].upload(np.full((rows, columns), 321, np.float16))
        first = {}
        for n in (1, 32, 33, 300, 448, 512, 513, 700):
            op.enqueue(n)
            first[n] = read(n)[:n]
        for n in (300, 700, 300):
            kw["output"].upload(np.full((rows, columns), 321, np.float16))
            op.enqueue(n)
            np.testing.assert_array_equal(read(n)[:n], first[n])
        start, end = abi.Event(ctx), abi.Event(ctx)
        op.enqueue(300, start=start, end=end)
        ctx.synchronize()
        assert 0 < start.elapsed_ms(end) < 1000
        start.destroy(), end.destroy()
        graph = abi.Graph.capture(ctx, ctx.stream)
        with graph:
            op.enqueue(300, ctx.stream)
        for n in (300, 64, 700):
            kw["output"].upload(np.full((rows, columns), 321, np.float16))
            op.enqueue(n)
            graph.launch()
            np.testing.assert_array_equal(read(max(n, 300))[:300], first[300])
    finally:
        if graph:
            graph.release()
        op.release()
