"""f16 attention where few tokens take nearly all: weights far below the largest.
A weight is rounded to f16 relative to a running maximum whose own weight is 2^7 at least, so
that one of p (the largest: 1) is off by 2^-11 of itself, or by 2^-25 / 2^7 = 2^-32 where that is more."""
import numpy as np
import pytest

from test_gpu_cache import attention_rows, run_attention, scope  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count,heads,kv_heads,dim", [(1, 4, 4, 64), (1, 2, 1, 128), (9, 4, 2, 64), (30, 2, 1, 40),
                                                      (140, 2, 1, 128)])
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
    cache, got, queries = run_attention(abi, ctx, scope, np.random.default_rng(1), np.float16, [count], [length], heads,
                                        kv_heads, dim, 16, scale=1.0, spoil=sink, check=False)
    want, size, slack, least = attention_rows(cache, queries, heads, scale=1.0)
    half = 2.0 ** -11
    weights = 2 * (dim + 4) * 2.0 ** -24 * slack + (8 + 4 * length ** 0.5) * 2.0 ** -24 + half
    bound = half * np.abs(want) + (1 + half) * (weights * size + least * 2.0 ** -32) + 2.0 ** -24
    off = np.abs(got.reshape(want.shape).astype(np.float64) - want) / bound
    assert off.max() <= 1, off.max()


@pytest.mark.parametrize("counts,heads,kv_heads,dim", [([1, 1], 2, 2, 64), ([7, 3], 4, 2, 128), ([50, 20], 2, 1, 64),
                                                       ([140, 90], 2, 1, 96), ([1, 2], 1, 1, 256)])
@pytest.mark.parametrize("length", [500, 3000])
@pytest.mark.parametrize("sign", [1, -1])
def test_values_of_the_largest_number(abi, ctx, scope, counts, heads, kv_heads, dim, length, sign):
    """A mean of f16's largest number is that number, and no infinity, also where nearly all weights are rounded
    up: of scores 0.00055 above those of the first tokens, by 0.00043."""
    largest = float(np.finfo(np.float16).max)

    def spoil(cache, queries):
        cache.values[:] = sign * largest
        queries[:] = 0
        queries[:, ::dim] = 1
        for s, n in enumerate(cache.lengths):
            for t in range(int(n)):
                for h in range(kv_heads):
                    cache.keys[cache.place(s, t) + h * 16 * dim] = 0.00055 if t >= 128 else 0
    cache, got, queries = run_attention(abi, ctx, scope, np.random.default_rng(dim), np.float16, counts, [length, 500],
                                        heads, kv_heads, dim, 16, scale=1.0, spoil=spoil, check=False)
    got = got.astype(np.float64)
    assert np.isfinite(got).all()
    # the weights' rounding, half a step, and the sums'
    assert (np.abs(got - sign * largest) <= largest * (2.0 ** -10 + 2.0 ** -16)).all()
