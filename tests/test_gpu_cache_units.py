"""Units of every kernel of the attention: 16, 32, 64 and 128 rows, heads of every width
class, whole and split, causal and not."""
import numpy as np
import pytest

from test_gpu_cache import DTYPES, run_attention, scope  # noqa: F401

pytestmark = pytest.mark.gpu


@DTYPES
@pytest.mark.parametrize("dim", [40, 64, 80, 96, 104, 128, 136, 192, 200, 256])
@pytest.mark.parametrize("count", [3, 13, 30, 70])  # 6 to 140 rows of a kv head
@pytest.mark.parametrize("length", [200, 1700])
def test_units(abi, ctx, scope, dtype, dim, count, length):
    rng = np.random.default_rng(dim * count)
    run_attention(abi, ctx, scope, rng, dtype, [count], [length], 4, 2, dim, 16)
    run_attention(abi, ctx, scope, rng, dtype, [count, count + 3, count], [length, 900, count], 2, 1, dim, 24, causal=False)
    run_attention(abi, ctx, scope, rng, dtype, [count], [length], 2, 1, dim, 8, window=600, cap=30.0)


@DTYPES
@pytest.mark.parametrize("count", [1, 5, 40])
def test_fewer_active_sequences(abi, ctx, scope, dtype, count):
    """The active sequences choose the rows of a unit: from 40 sequences down to one."""
    rng = np.random.default_rng(count)
    lengths = [int(x) for x in rng.integers(count, 900, 40)]
    for active in (1, 2, 7, 20, 39):
        run_attention(abi, ctx, scope, rng, dtype, [count] * 40, lengths, 4, 1, 64, 16, active=active)
