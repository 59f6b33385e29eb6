"""Rows before position 0, of sequences that are shorter than their rows. With causality
they see nothing and give zeros, beside rows of the same block that see something; without, a
row's position does not matter, and these see what the sequence holds, as all its rows do."""
import numpy as np
import pytest

from test_gpu_cache import DTYPES, attention_rows, check_attention, run_attention, scope  # noqa: F401

pytestmark = pytest.mark.gpu


@DTYPES
@pytest.mark.parametrize("count,length", [(3, 1), (4, 0), (30, 20), (40, 39), (120, 50), (300, 200)])
@pytest.mark.parametrize("dim", [64, 128, 200])
def test_rows_before_position_zero(abi, ctx, scope, dtype, count, length, dim):
    run = lambda **kw: run_attention(abi, ctx, scope, np.random.default_rng(count), dtype, [count, 2], [count, 30], 4, 2,
                                     dim, 16, **kw)

    def spoil(cache, queries):
        cache.lengths[0] = length
    cache, got, queries = run(spoil=spoil, causal=False)
    assert not length or (got[:count] != 0).any(axis=1).all()
    cache, got, queries = run(spoil=spoil, causal=True)
    assert (got[:count - length] == 0).all()
    cache, got, queries = run(spoil=spoil, causal=True, window=7)
    assert (got[:count - length] == 0).all()

    def strange(cache, queries):  # a value that only the later rows see does not reach those before
        spoil(cache, queries)
        at = cache.place(0, 0)
        if length:
            cache.values[at] = np.inf
    cache, got, queries = run(spoil=strange, causal=True, check=False)
    assert (got[:count - length] == 0).all()
    if length:
        got = got.reshape(len(got), 4, dim).copy()
        assert (got[count - length:count, :2, 0] == np.inf).all()  # both heads of kv head 0
        cache.values[cache.place(0, 0)] = 0
        want = attention_rows(cache, queries, 4)[0]
        got[count - length:count, :2, 0] = want[count - length:count, :2, 0].astype(dtype)
        check_attention(cache, got.reshape(len(got), -1), queries, 4)
