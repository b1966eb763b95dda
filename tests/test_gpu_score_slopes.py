"""Slopes at the end of f32's range: a bias that would be infinite is refused, one that is
not chooses the nearest or the farthest key alone, and a sum that is not finite is reported."""

import numpy as np
import pytest

import test_gpu_score as ts
from tvara_amd import _capi

pytestmark = pytest.mark.gpu
SHAPES = [(64, 1), (128, 1), (64, 170), (128, 170), (96, 3)]


@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
@pytest.mark.parametrize("dim,count", SHAPES)
def test_the_largest_slopes(device, oracle, dim, count, fmt):
    ts.say("score, large slopes", dim, count, fmt)
    n = 200
    b = ts.Batch(device, oracle, 2, 2, dim, [n], [count], q8=fmt == "q8_0")
    for bad in (1e38, -1e38, 3e35, -3e35, 2.3e38):
        for slopes in ([0.0, bad], [bad, bad]):
            with pytest.raises(_capi.InvalidArgument, match="slope"):
                b.run(slopes=slopes)
    # keys well before a row's own place, and for the last rows behind it: f32's spacing there is
    # 2e28, so that the nearest key, or the farthest, has all the weight
    end = np.full(count, 20)
    first = np.full(count, 4)
    got = b.run(first=first, end=end, slopes=[2.9e35, -2.9e35]).reshape(count, 2, dim)
    place = n - count + np.arange(count)
    near, far = np.clip(place, 4, 19), np.where(abs(place - 4) >= abs(place - 19), 4, 19)
    v = b.v[0].reshape(n, 2, dim)
    alone = abs(place - 4) != abs(place - 19)
    # (a value in two fp16 parts is off by 2^-23)
    assert np.allclose(got[:, 0], v[near, 0], rtol=2.0 ** -22, atol=1e-7)
    assert np.allclose(got[alone, 1], v[far, 1][alone], rtol=2.0 ** -22, atol=1e-7)


@pytest.mark.parametrize("dim,count", SHAPES)
def test_a_sum_that_is_not_finite_is_reported(device, oracle, dim, count):
    """A score just inside f32 and a bias that takes it out."""
    ts.say("score, score and bias", dim, count)
    n = 200

    def poison(i, k, v):
        k[:] = 0
        k[0, 0] = 2.0 ** 60
        return k, v

    b = ts.Batch(device, oracle, 1, 1, dim, [n], [count], poison=poison)
    b.q[:] = 0
    b.q[:, 0] = 1.3 * 2.0 ** 67  # a score of 3.2e38 in log2 units
    with pytest.raises(_capi.InvalidArgument, match="invalid online attention input"):
        b.run(scale=1.0, slopes=[-2.9e35], first=np.zeros(count, int), end=np.full(count, n))
