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
