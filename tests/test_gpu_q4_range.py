"""The range of the 4-bit product's sums (pk_q4): activations whose magnitudes
add up to less than 2^125 over a group give the formula's outputs, and larger
or infinite ones give outputs that are no numbers, in their own rows alone."""
import numpy as np
import pytest

import test_gpu_q4 as q4
from test_gpu_parity import Scope

pytestmark = pytest.mark.gpu


@pytest.fixture
def scope(ctx):
    s = Scope(ctx)
    yield s
    s.close()


@pytest.mark.parametrize("offsets", [False, True])
@pytest.mark.parametrize("rows", [1, 3, 20, 700])
def test_large_f32_activations(abi, ctx, scope, rows, offsets):
    case = q4.make(np.random.default_rng(rows), np.float32, rows, 300, 2064, 64, offsets)
    case["scales"] = case["scales"] * np.float32(2.0 ** -100)
    if offsets:
        case["offsets"] = case["offsets"] * np.float32(2.0 ** -100)
    unit = case["a"]
    sums = np.add.reduceat(np.abs(unit.astype(np.float64)), np.arange(0, 300, 64), axis=1)
    case["a"] = (unit * np.float32(2.0 ** 124.9 / sums.max())).astype(np.float32)
    clean = q4.run(abi, ctx, scope, case)
    q4.check(clean, case)
    # half of the largest number in 16 places of a group: its sums pass the range whatever the codes but 8
    case["a"][rows // 2, 64:80] = 2.0 ** 127
    case["codes"][64:80] = np.maximum(case["codes"][64:80], 9)
    plain = q4.run(abi, ctx, scope, case)
    assert not np.isfinite(plain[rows // 2]).any()
    case["a"][rows // 2, 64:80] = unit[rows // 2, 64:80]
    q4.check(q4.run(abi, ctx, scope, case), case)  # the other codes, without those activations
    others = [r for r in range(rows) if r != rows // 2]
    want, tol = q4.reference(case)
    assert (np.abs(plain[others].astype(np.float64) - want[others]) <= tol[others]).all()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows", [1, 3, 20, 700])
def test_an_infinite_activation_with_offsets(abi, ctx, scope, dtype, rows):
    """Infinities or NaN (the formula has infinities): the group's sum of codes
    and its sum for the offset may be opposite infinities."""
    case = q4.make(np.random.default_rng(rows), dtype, rows, 300, 2064, 64, True)
    clean = q4.run(abi, ctx, scope, case)
    case["a"][rows // 2, 70] = -np.inf
    got = q4.run(abi, ctx, scope, case)
    others = [r for r in range(rows) if r != rows // 2]
    np.testing.assert_array_equal(got[others], clean[others])
    assert not np.isfinite(got[rows // 2]).any()
