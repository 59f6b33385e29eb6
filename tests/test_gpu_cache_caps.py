"""Score caps far above the scores: cap * tanh(z / cap) is then nearly z, and what
tanh is off by counts cap times. Of a capped score 2^-19 is granted, relative to it: 1 - 2 / (1 +
e^2x) is within 2^-21 from x = 1/4 on, where tanh is 1/4, and a series relative to x below.
Caps of up to 256 may be off by 2^-23 of the cap instead, a tenth of what the weights'
rounding to f16 is."""
import numpy as np
import pytest

from test_gpu_cache import DTYPES, HALF_STEP, attention_rows, run_attention, scope  # noqa: F401

pytestmark = pytest.mark.gpu


def check_capped(cache, got, queries, heads, cap, longest):
    want, size, slack, least = attention_rows(cache, queries, heads, cap=cap)
    half = HALF_STEP[cache.dtype]
    capped = cap * np.tanh(slack / cap)
    score = (cache.dim + 4) * 2.0 ** -24 * slack + 2.0 ** -19 * capped + (2.0 ** -22 * cap if cap <= 256 else 0)
    weights = 2 * score + (8 + longest ** 0.5 * 4) * 2.0 ** -24 + (2.0 ** -11 if cache.dtype == np.float16 else 0)
    bound = half * np.abs(want) + (1 + half) * (weights * size + least * (2.0 ** -25 if cache.dtype == np.float16 else 0))
    bound = bound + np.finfo(cache.dtype).smallest_subnormal
    off = np.abs(got.reshape(want.shape).astype(np.float64) - want) / bound
    assert off.max() <= 1, (off.max(), np.argwhere(off > 1)[:4])


@DTYPES
@pytest.mark.parametrize("counts", [[1, 1], [9, 4], [70, 40], [140, 100]])
@pytest.mark.parametrize("cap", [1.0, 50.0, 256.0, 257.0, 4096.0, 65536.0, 2.0 ** 20])
@pytest.mark.parametrize("std", [0.1, 2.0, 30.0])
def test_large_caps(abi, ctx, scope, dtype, counts, cap, std):
    cache, got, queries = run_attention(abi, ctx, scope, np.random.default_rng(int(cap)), dtype, counts, [300, 150], 2, 1,
                                        128, 16, cap=cap, query_std=std, check=False)
    check_capped(cache, got, queries, 2, cap, 300)


@DTYPES
@pytest.mark.parametrize("count", [2, 13, 30, 70])  # units of 16, 32, 64 and 128 rows
@pytest.mark.parametrize("dim", [40, 64, 80, 128, 192, 256])
def test_large_caps_of_every_unit(abi, ctx, scope, dtype, count, dim):
    cap = 65536.0
    cache, got, queries = run_attention(abi, ctx, scope, np.random.default_rng(dim), dtype, [count, 1], [1200, 150], 4, 2,
                                        dim, 16, cap=cap, check=False)
    check_capped(cache, got, queries, 4, cap, 1200)
