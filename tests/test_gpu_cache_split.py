"""Sequences that are split over workgroups: units of every size and head width,
and infinities and NaN in the parts."""
import numpy as np
import pytest

from test_gpu_cache import DTYPES, attention_rows, check_attention, run_attention, scope  # noqa: F401

pytestmark = pytest.mark.gpu


@DTYPES
@pytest.mark.parametrize("strange", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("count,heads,kv_heads,dim", [(1, 2, 1, 64), (1, 1, 1, 256), (6, 4, 1, 64), (30, 2, 2, 128),
                                                      (60, 1, 1, 40), (140, 2, 1, 128)])
@pytest.mark.parametrize("length", [1500, 5000])
def test_infinities_in_a_part(abi, ctx, scope, dtype, strange, count, heads, kv_heads, dim, length):
    """One channel of the newest token's values is not finite: the last row has it there, all else
    is what it would be."""
    def newest(cache, queries):
        for h in range(kv_heads):
            cache.values[cache.place(0, length - 1) + h * 16 * dim + 5] = strange
    cache, got, queries = run_attention(abi, ctx, scope, np.random.default_rng(dim), dtype, [count], [length], heads,
                                        kv_heads, dim, 16, query_std=0.5, spoil=newest, check=False)
    got = got.reshape(count, heads, dim).copy()
    np.testing.assert_array_equal(got[-1, :, 5], np.full(heads, strange, dtype))
    for h in range(kv_heads):
        cache.values[cache.place(0, length - 1) + h * 16 * dim + 5] = 0
    got[-1, :, 5] = attention_rows(cache, queries, heads)[0][-1, :, 5].astype(dtype)
    check_attention(cache, got.reshape(count, -1), queries, heads)
