"""What the product with 4-bit weights (pk_q4) keeps of its operands' digits.

Whole numbers: activations are whole and scales and offsets whole multiples of
one power of two, so small that every sum of their products stays below 2^24 of
that unit. No f32 addition rounds then, in whatever order, and an output is the
exact sum rounded once: what a lane reads before another has written it, a sum
held in fewer bits or an operand rounded to them is off by whole units."""
import numpy as np
import pytest

import test_gpu_q4 as q4
from test_gpu_parity import Scope

UNIT = 2.0 ** -9


@pytest.fixture
def scope(ctx):
    s = Scope(ctx)
    yield s
    s.close()


def whole(rng, dtype, rows, inner, columns, group, offsets):
    """A case of whole numbers, and its exact outputs in float64."""
    case = q4.make(rng, dtype, rows, inner, columns, group, offsets, bias=True)
    shape = case["scales"].shape
    a = rng.integers(-1, 2, (rows, inner))
    if dtype == np.float32:  # some of 13 bits: f16 holds 11
        at = rng.integers(0, inner, (rows, 8))
        a[np.arange(rows)[:, None], at] = rng.integers(2048, 4096, at.shape) * 2 + 1
    case["a"] = a.astype(dtype)
    case["scales"] = (rng.integers(1, 3, shape) * UNIT).astype(dtype)
    if offsets:
        case["offsets"] = (rng.integers(-3, 4, shape) * UNIT).astype(dtype)
    case["bias"] = (rng.integers(-99, 100, columns) * UNIT).astype(np.float32)
    at = np.arange(inner) // (group or inner)
    scale, offset = case["scales"].astype(np.float64)[at], case["offsets"].astype(np.float64)[at] if offsets else 0.0
    w = scale * (case["codes"].astype(np.float64) - 8) + offset
    # every partial sum of products and of offsets, whatever its order
    assert (np.abs(a).astype(np.float64) @ (np.abs(scale * 8) + np.abs(offset))).max() + 99 * UNIT < 2 ** 24 * UNIT
    return case, case["a"].astype(np.float64) @ w + case["bias"]


@pytest.mark.gpu
@pytest.mark.parametrize("offsets", [False, True])
@pytest.mark.parametrize("dtype,rows,inner,columns,group", [
    # workgroups of 16 rows x 16 columns, 16 x 32, 32 x 32 and 64 x 32, whose wavefronts take several blocks of K each
    (np.float16, 20, 9000, 64, 64), (np.float16, 40, 4224, 2100, 128), (np.float16, 24, 2600, 4100, 32),
    (np.float16, 60, 4100, 6600, 64),
    (np.float32, 6, 9000, 64, 128), (np.float32, 20, 4100, 500, 32), (np.float32, 48, 2304, 1000, 64)])
def test_rows_copied_by_their_wavefronts(abi, ctx, scope, dtype, rows, inner, columns, group, offsets):
    """A wavefront's lanes read rows that others of its lanes copied, block after
    block through one area: to the bit, several times over."""
    case, want = whole(np.random.default_rng(rows + inner), dtype, rows, inner, columns, group, offsets)
    kw = q4.operands(abi, scope, case)
    op = abi.Q4GemmOp(ctx, **kw)
    try:
        for _ in range(3):
            op.enqueue()
            ctx.synchronize()
            np.testing.assert_array_equal(kw["output"].download(), want.astype(dtype))
    finally:
        op.release()


@pytest.mark.gpu
@pytest.mark.parametrize("offsets", [False, True])
@pytest.mark.parametrize("dtype,rows,inner,columns,group", [
    # parts of K that meet in a workspace, tiles whole, rows whole in LDS
    (np.float16, 500, 17300, 512, 128), (np.float16, 130, 4100, 5500, 64), (np.float16, 64, 8192, 8200, 32),
    (np.float16, 700, 1100, 2100, 0), (np.float16, 16, 2300, 300, 32), (np.float16, 1, 12000, 100, 128),
    (np.float32, 500, 4200, 512, 128), (np.float32, 130, 1100, 5500, 64), (np.float32, 700, 600, 2100, 32),
    (np.float32, 5, 1100, 300, 64), (np.float32, 4, 2300, 100, 32), (np.float32, 1, 12000, 100, 0)])
def test_whole_numbers(abi, ctx, scope, dtype, rows, inner, columns, group, offsets):
    case, want = whole(np.random.default_rng(rows * 3 + inner), dtype, rows, inner, columns, group, offsets)
    np.testing.assert_array_equal(q4.run(abi, ctx, scope, case), want.astype(dtype))


# The f32 sizes of test_gpu_q4's long axes, row counts, tiles and parts of K.
F32 = [(rows, inner, columns, 64, False, False) for rows in (1, 20)
       for inner, columns in ((4096, 64), (64, 4096), (8192, 16), (2560, 2560), (9000, 129))] + \
      [(rows, 1024, 520, 128, True, False) for rows in (1, 2, 4, 5, 8, 9, 31, 32, 48, 100, 257)] + \
      [(640, 300, 2100, 64, True, False), (1504, 128, 1032, 0, False, False), (800, 260, 1700, 128, False, False),
       (500, 4200, 512, 128, False, True), (130, 1100, 5500, 64, True, True), (49, 8192, 2050, 32, True, True)]


def f32_case(rows, inner, columns, group, offsets, epilogue):
    more = dict(activation="silu", residual=True, residual_scale=2.0) if epilogue else {}
    return q4.make(np.random.default_rng(rows * inner + columns), np.float32, rows, inner, columns, group, offsets,
                   bias=True, **more)


def f32_reference(case, a=None, parts=1, cast=np.float64, weight=np.float64):
    """(outputs, tolerance) in float64; with other activations, with the weight
    of another type, or with the sum over K as that many parts of type `cast`."""
    inner, columns = case["codes"].shape
    at = np.arange(inner) // (case["group_size"] or inner)
    scaled = case["scales"].astype(np.float64)[at] * (case["codes"].astype(np.float64) - 8)
    offset = case["offsets"].astype(np.float64)[at] if "offsets" in case else np.zeros((1, columns))
    w = (scaled + offset).astype(weight).astype(np.float64)
    x = (case["a"] if a is None else a).astype(np.float64)
    ends = np.linspace(0, inner, parts + 1).astype(int)
    v = sum((x[:, i:j] @ w[i:j]).astype(cast).astype(np.float64) for i, j in zip(ends, ends[1:]))
    squares = x ** 2
    size = np.sqrt(squares @ (scaled ** 2) + (squares @ np.broadcast_to(offset ** 2, w.shape)))
    tol = 12 * 2.0 ** -24 * np.sqrt(inner) * size
    v = v + case["bias"]
    tol = tol + 2.0 ** -24 * np.abs(v)
    if case["activation"] == "silu":
        y = v / (1 + np.exp(-v))
        tol, v = 1.1 * tol + (np.abs(v) + 4) * 2.0 ** -23 * np.abs(y), y
    if "residual" in case:
        v = case["residual"] + case["residual_scale"] * v
        tol = abs(case["residual_scale"]) * tol + 2.0 ** -23 * np.abs(v)
    return v, tol + 2.0 ** -24 * np.abs(v) + 2.0 ** -149


@pytest.mark.parametrize("size", F32)
def test_what_the_f32_tolerance_rejects(size):
    """It takes an f32 product, and neither f16 operands nor parts of sums in f16."""
    case = f32_case(*size)
    want, tol = f32_reference(case)
    inner = size[1]

    def worst(**other):
        return (np.abs(f32_reference(case, **other)[0] - want) / tol).max()
    assert worst(a=case["a"].astype(np.float16)) > 2
    assert worst(weight=np.float16) > 2
    assert worst(parts=min(8, inner // 32), cast=np.float16) > 2
    at = np.arange(inner) // (case["group_size"] or inner)
    w = case["scales"][at] * (case["codes"].astype(np.float32) - 8)
    if "offsets" in case:
        w = w + case["offsets"][at]
    plain = dict(case, activation="none")
    plain.pop("residual", None)
    v, v_tol = f32_reference(plain)
    assert (np.abs((case["a"] @ w).astype(np.float64) + case["bias"] - v) <= v_tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("size", F32)
def test_f32_products_keep_their_digits(abi, ctx, scope, size):
    case = f32_case(*size)
    want, tol = f32_reference(case)
    got = q4.run(abi, ctx, scope, case).astype(np.float64)
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()
