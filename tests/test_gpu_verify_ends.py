"""Draft verification at the ends of its ranges: rows whose first and last parts
are masked whole, and draws that end there."""
import numpy as np
import pytest

import test_gpu_verify as verify
from test_gpu_verify import DTYPES, scope  # noqa: F401

pytestmark = pytest.mark.gpu

ENDS = [0.0, -1.0, 1.0, np.nan, 2.0, -np.inf, np.inf, 0.5]


def single_rows(rng, dtype, sequences, columns, rows_each=1):
    """Sequences of rows that have no draft: each draws from its first."""
    case = verify.make(rng, dtype, [rows_each] * sequences, columns, drafted=False)
    case["tokens"][:] = verify.NO_TOKEN
    return case


@DTYPES
@pytest.mark.parametrize("columns,rows_each", [(600, 1), (3000, 20), (20000, 1), (40000, 2)])
@pytest.mark.parametrize("lowest", [False, True])
@pytest.mark.parametrize("residual", [False, True])
def test_masked_parts(abi, ctx, scope, dtype, columns, rows_each, lowest, residual):
    """At a last row, and after a refusal where the target is nowhere above the draft."""
    rng = np.random.default_rng(columns)
    case = single_rows(rng, dtype, len(ENDS), columns, max(rows_each, 2 if residual else 1))
    low = np.finfo(dtype).min if lowest else -np.inf
    first, last = int(columns * 0.45), int(columns * 0.6)
    case["target"][:, :first] = low
    case["target"][:, last:] = low
    case["draws"][:] = ENDS
    if residual:
        case["draft"] = case["target"].copy()
        case["tokens"][:] = first + 5
        case["uniforms"][:] = 2.0
    want = verify.check(abi, ctx, scope, case)
    assert (want[0] == 0).all() and ((want[1] >= first) & (want[1] < last)).all()
    assert want[1][0] == first and want[1][2] == last - 1


@DTYPES
@pytest.mark.parametrize("columns", [70, 1025, 4096, 20000, 131072])
def test_draws_from_one_on(abi, ctx, scope, dtype, columns):
    """The last token with a weight, be that far below the sum's last digit."""
    rng = np.random.default_rng(columns)
    case = single_rows(rng, dtype, 48, columns)
    case["target"][:, -1] = -45
    case["target"][::3, columns // 2 + 1:] = -40
    case["draws"][:] = np.resize(np.array([1.0, np.nan, 2.0, np.inf], np.float32), 48)
    want = verify.check(abi, ctx, scope, case)
    assert (want[1] == columns - 1).all()


@pytest.mark.parametrize("columns", [100, 9000])
def test_probabilities_that_count_as_zero(abi, ctx, scope, columns):
    """Below 2^-990: a draft of that probability is refused, even by a uniform of 0, and is not drawn."""
    case = verify.make(np.random.default_rng(1), np.float32, [2, 2], columns, drafted=False)
    case["target"][:] = -1e30
    case["target"][:, 7] = 0
    case["target"][0, 50] = -685          # 2^-988
    case["target"][2, 50] = -690          # 2^-995
    case["tokens"][:] = 50
    case["uniforms"][:] = 0
    case["draws"][:] = [1.0, 1.0]
    got = verify.run(abi, ctx, scope, case)
    assert list(got[0]) == [1, 0]
    assert list(got[1]) == [7, 7]
