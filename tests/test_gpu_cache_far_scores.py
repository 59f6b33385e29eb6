"""Scores far beyond 2^24, where a step of f32 is more than one: the products are
whole numbers times a power of two, exact, and their gaps many steps, so that the largest takes all,
equal ones share, and nothing overflows."""
import numpy as np
import pytest

from test_gpu_cache import DTYPES, attention_rows, run_attention, scope  # noqa: F401

pytestmark = pytest.mark.gpu


@DTYPES
@pytest.mark.parametrize("counts,heads,kv_heads,dim,length", [
    ([1], 2, 1, 64, 300), ([1], 1, 1, 128, 3000), ([9], 4, 2, 64, 300), ([70], 2, 1, 128, 300), ([140], 2, 1, 128, 2000),
    ([20], 1, 1, 256, 200)])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("exponent", [0, 8, 12, 16, 20, 24, 40, 59])
def test_far_scores(abi, ctx, scope, dtype, counts, heads, kv_heads, dim, length, sign, exponent):
    """sign -1: all scores far below zero."""
    rng = np.random.default_rng(exponent)
    order = rng.permutation(length)

    def spoil(cache, queries):
        queries[:] = 0
        queries[:, ::dim] = 1000 + np.arange(len(queries))[:, None]
        for h in range(kv_heads):
            for t in range(length):
                cache.keys[cache.place(0, t) + h * 16 * dim] = sign * (1 + order[t] // 2)  # two of each
    half = 2.0 ** -11 if dtype == np.float16 else 2.0 ** -24
    for step in range(8):  # the maxima round up and down
        scale = float(np.float32(2.0 ** exponent * (1 + step / 9)))
        cache, got, queries = run_attention(abi, ctx, scope, rng, dtype, counts, [length], heads, kv_heads, dim, 16,
                                            scale=scale, spoil=spoil, check=False)
        want, size, slack, least = attention_rows(cache, queries, heads, scale=scale)
        # equal scores have equal weights; others' are 0, as a gap is 1000 at least
        bound = half * np.abs(want) + 4 * half * size + 2.0 ** -24
        off = np.abs(got.reshape(want.shape).astype(np.float64) - want) / bound
        assert np.isfinite(off).all() and off.max() <= 1, (scale, off.max())
