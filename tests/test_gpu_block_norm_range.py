"""The range of the norms around a block (pk_block_norm) in f32: numbers whose
squares add up within it, with the tolerances of test_gpu_block_norm."""
import numpy as np
import pytest

import test_gpu_block_norm as norm
from test_gpu_parity import Scope

pytestmark = pytest.mark.gpu


@pytest.fixture
def scope(ctx):
    s = Scope(ctx)
    yield s
    s.close()


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("channels", [40, 1025, 16384])
@pytest.mark.parametrize("top,epsilon", [(2.0 ** 56, None), (2.0 ** -50, 0.0)])
def test_large_and_small_f32_rows(abi, ctx, scope, channels, kind, post, top, epsilon):
    """Rows whose largest magnitude lies just below 2^56, and, without an
    epsilon to drown them in, rows of 2^-50."""
    case = norm.make(np.random.default_rng(channels), np.float32, 5, channels, kind, "none", post, epsilon=epsilon)
    for name in ("input", "residual"):
        a = case[name].astype(np.float64)
        case[name] = (a * (0.99 * top / np.abs(a).max())).astype(np.float32)
    if not post:  # the sum of both feeds the norm
        case["residual"] = case["residual"] / np.float32(2)
    norm.check(norm.run(abi, ctx, scope, case), case)
