"""f16 attention where few tokens take nearly all: weights far below the largest.
A weight is rounded to f16 relative to a running maximum whose own weight is 2^7 at least, so
that one of p (the largest: 1) is off by 2^-11 of itself, or by 2^-25 / 2^7 = 2^-32 where that is more."""
import numpy as np
import pytest

from test_gpu_cache import attention_rows, run_attention, scope  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count,heads,kv_heads,dim", [(1, 4, 4, 64), (1, 2, 1, 128), (9, 4, 2, 64), (30, 2, 1, 40), (140, 2, 1, 128)])
@pytest.mark.parametrize("gap", [10.0, 14.0, 16.0, 17.0, 17.5])
@pytest.mark.parametrize("rising", [False, True])
def test_small_weights(abi, ctx, scope, count, heads, kv_heads, dim, gap, rising):
    """A first token without a value of its own, `gap` above all others; then the same where scores
    rise to it in steps, so that the maximum follows."""
    length = 500 if count == 1 else 400

    def sink(cache, queries):
        queries[:] = 0
        queries[:, ::dim] = 1
        for h in range(kv_heads):
            for t in range(length):
                at = cache.place(0, t) + h * 16 * dim
                cache.keys[at] = min(t // 32 * 0.75, gap / 2) if rising else 0
                cache.values[at:at + dim] = 1000 + np.arange(dim)
            at = cache.place(0, 0) + h * 16 * dim
            cache.keys[at] = gap
            cache.values[at:at + dim] = 0
    cache, got, queries = run_attention(abi, ctx, scope, np.random.default_rng(1), np.float16, [count], [length], heads, kv_heads,
                                        dim, 16, scale=1.0, spoil=sink, check=False)
    want, size, slack, least = attention_rows(cache, queries, heads, scale=1.0)
    half = 2.0 ** -11
    weights = 2 * (dim + 4) * 2.0 ** -24 * slack + (8 + 4 * length ** 0.5) * 2.0 ** -24 + half
    bound = half * np.abs(want) + (1 + half) * (weights * size + least * 2.0 ** -32) + 2.0 ** -24
    off = np.abs(got.reshape(want.shape).astype(np.float64) - want) / bound
    assert off.max() <= 1, off.max()
