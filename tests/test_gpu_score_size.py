"""Scores of any size that f32 holds: beside one far above the others its value is the
output, whichever kernel a row takes."""

import numpy as np
import pytest

import test_gpu_score as ts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cap", [0.0, 1e15])
@pytest.mark.parametrize("power", [8, 15, 20, 25, 31, 40, 64, 100, 126])
@pytest.mark.parametrize("dim,count", [(64, 1), (128, 1), (64, 170), (128, 170), (96, 3)])
def test_large_scores(device, oracle, dim, count, power, cap):
    """Rows of scores that differ in all their bits, with one key an eighth of them above the
    others; far above a cap all are equal."""
    ts.say("score, large scores", dim, count, power, cap)
    n = 200
    rng = np.random.default_rng(power)

    def poison(i, k, v):
        k[:] = 0
        k[:, 0] = 2.0 ** (power // 2) * (1 + 0.25 * rng.random(n))
        k[50, 0] = 2.0 ** (power // 2) * 1.4
        return k, v

    b = ts.Batch(device, oracle, 1, 1, dim, [n], [count], poison=poison)
    b.q[:] = 0
    b.q[:, 0] = 2.0 ** (power - power // 2) * (0.85 + 0.15 * rng.random(count)) / 1.4427
    got = b.run(scale=1.0, cap=cap, first=np.zeros(count, int), end=np.full(count, n))
    s = b.q[:, :1].astype(np.float64) @ b.k[0][:, :1].astype(np.float64).T
    if cap:
        s = cap * np.tanh(s / cap)
    w = np.exp(s - s.max(1, keepdims=True))
    want = w @ b.v[0].astype(np.float64) / w.sum(1, keepdims=True)
    # the others' weights are e^-(2^power / 12) of the largest, 5e-10 at 2^8 and nothing beyond, or
    # 1: values, weights and sums are off by 2^-21 and 2^-19 of what is added up at the most
    assert np.allclose(got, want, rtol=2.0 ** -21, atol=4e-6)


@pytest.mark.parametrize("cap", [1e18, 1e20, 1e30, 1e35, 2e38])
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
@pytest.mark.parametrize("dim,count", [(64, 1), (128, 1), (64, 170), (128, 170), (96, 3)])
def test_large_caps(device, oracle, dim, count, fmt, cap):
    """Caps far above every score change none: the bars are those without a cap."""
    ts.say("score, large caps", dim, count, fmt, cap)
    b = ts.Batch(device, oracle, 2, 1, dim, [200], [count], q8=fmt == "q8_0")
    b.agree(b.run(cap=cap))
