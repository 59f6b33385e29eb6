"""Token scores (pk_score) of f32 logits that lie further apart than the largest
f32: with a temperature above one their log probabilities are numbers again.
Against float64, with the tolerances of test_gpu_score."""
import numpy as np
import pytest

import test_gpu_score as score
from test_gpu_parity import Scope

pytestmark = pytest.mark.gpu


@pytest.fixture
def scope(ctx):
    s = Scope(ctx)
    yield s
    s.close()


@pytest.mark.parametrize("temperature", [1.0, 1.5, 4.0, 2.0 ** 20, 0.5])
@pytest.mark.parametrize("columns", [5, 300, 2000, 140001])
def test_logits_of_both_ends(abi, ctx, scope, columns, temperature):
    """The lowest number as a mask below logits so large that their difference
    is none, as a given token and as an alternative."""
    low, high = np.finfo(np.float32).min, np.finfo(np.float32).max
    logits = np.full((6, columns), low, np.float32)
    logits[0, 1] = high
    logits[1, :2] = high, high / 2
    logits[2, 3] = 2.0 ** 104  # half a step of the lowest number
    logits[3, 2] = 1.0
    with np.errstate(over="ignore"):
        logits[4, 1:] = np.random.default_rng(columns).standard_normal(columns - 1) * 1e38
    logits[5, 0] = -high / 2
    tokens = np.array([0, 1, 4, 0, 0, 3], np.uint32)
    got = score.run(abi, ctx, scope, logits, tokens, 4, temperature=temperature)
    score.check(got, logits, tokens, 4, temperature)
    if temperature == 4.0:
        plain = np.isfinite(logits).all(1)  # the random row has numbers beyond f32, thus infinities, in some sizes
        assert np.isfinite(got[0][plain]).all() and np.isfinite(got[3][plain]).all() and got[0][0] < -1e38
