"""Rotations by angles of up to 2^68 radians: the product of position and
frequency is reduced by whole turns before it is rounded."""
from fractions import Fraction

import numpy as np
import pytest

import test_gpu_cache as cache_test
from test_gpu_cache import DTYPES, HALF_STEP, scope  # noqa: F401

pytestmark = pytest.mark.gpu

TURN = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")


@DTYPES
@pytest.mark.parametrize("kind", ["halves", "neighbours"])
def test_large_frequencies(abi, ctx, scope, dtype, kind):
    rng = np.random.default_rng(1)
    frequencies = np.array([2.0 ** 36, -2.0 ** 36, 3.7e9, -1234567.9, 2.0 ** 20 + 0.125, 1.0, 1e-30, 0], np.float32)
    dim, rows = 16, 9
    positions = np.array([0, 1, 3, 2 ** 20 + 7, 2 ** 31 - 1, 2 ** 31, 2 ** 32 - 1, 4003210987, 3333333333], np.uint32)
    cache = cache_test.Cache(rng, dtype, [rows], [rows], 1, dim, 16)
    keys, values = (rng.standard_normal((rows, dim)).astype(dtype) for _ in range(2))
    op = abi.CacheAppendOp(ctx, keys=scope.put(keys), values=scope.put(values), rotary_dim=dim, rotary=kind,
                           frequencies=scope.put(frequencies), positions=scope.put(positions), **cache.put(scope))
    op.enqueue()
    ctx.synchronize()
    op.release()
    got = cache.device["key_cache"].download()
    for r, p in enumerate(positions):
        angle = np.array([float(Fraction(int(p)) * Fraction(float(f)) % TURN) for f in frequencies])
        exact, size = cache_test.rotate(keys[r][None], angle, kind)
        at = cache.place(0, r)
        bound = HALF_STEP[dtype] * np.abs(exact[0]) + 2.0 ** -22 * size[0] + np.finfo(dtype).smallest_subnormal
        assert (np.abs(got[at:at + dim].astype(np.float64) - exact[0]) <= bound).all(), p
