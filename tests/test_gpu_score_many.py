"""What rows do not see, and what is not finite, in the kernels of many rows and of few over
both layouts; each test says which kernel it is for."""

import numpy as np
import pytest

import test_gpu_score as ts
from tvara_amd import _capi, attention

pytestmark = pytest.mark.gpu
# appends encode a NaN among finite numbers as one of their bytes: of Q8_0 blocks only infinite
# scales are not finite
STORED = [("f32", np.inf), ("f32", np.nan), ("q8_0", np.inf)]
CASES = [("score_attention_shared", 170), ("score_attention_tiles", 1), ("score_attention_tiles", 40)]


def run(b, kernel, **how):
    attention.profile_reset()
    attention.profile_enable(True)
    try:
        got = b.run(**how)
        for name in ("score_attention_shared", "score_attention_tiles", "score_attention"):
            assert attention.profile_read(name)[1] == int(name == kernel), name
    finally:
        attention.profile_enable(False)
    return got.reshape(b.rows, b.heads, b.dim)


@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kernel,count", CASES)
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan, 3.4e38])
@pytest.mark.parametrize("style", [{}, {"cap": 7.0}, {"slopes": [0.1, 0.02]}])
def test_what_a_row_does_not_see_never_reaches_it(device, oracle, style, bad, kernel, count, dim, fmt):
    ts.say("score, unseen", kernel, count, bad, dim, fmt, style)
    if fmt == "q8_0" and bad == 3.4e38:
        bad = 1e30  # (its scale is infinite)
    n, hidden = 400, [0, 3, 40, 41, 177, 399]

    def poison(i, k, v):
        k[hidden], v[hidden] = bad, bad
        return k, v

    b = ts.Batch(device, oracle, 2, 2, dim, [n], [count], q8=fmt == "q8_0", poison=poison)
    gaps = [(4, 40), (42, 177), (178, n - 1), (1, 3), (5, 5), (190, 340)]
    how = {e: np.array([gaps[j % 6][i] for j in range(count)]) for i, e in enumerate(("first", "end"))}
    for x in (b.k, b.v):
        x[0] = np.nan_to_num(x[0], nan=0, posinf=0, neginf=0)  # (the 64-bit form multiplies ranges only)
    b.agree(run(b, kernel, **how, **style).reshape(count, -1), **how, **style)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kernel,count", CASES)
@pytest.mark.parametrize("fmt,bad", STORED)
def test_a_value_that_is_not_finite_shows(device, oracle, bad, kernel, count, dim, fmt):
    """In its column (of Q8_0: its group's) of the rows that see it, and nowhere else."""
    ts.say("score, not finite", kernel, count, bad, dim, fmt)
    holes = [(20, dim + 7), (100, 3), (301, 2 * dim - 1)]

    def poison(i, k, v):
        for at in holes:
            v[at] = bad
        return k, v

    b = ts.Batch(device, oracle, 2, 2, dim, [400], [count], q8=fmt == "q8_0", poison=poison)
    first = np.where(np.arange(count) % 2, 21, 0)
    end = np.where(np.arange(count) % 3, 330, 90)
    got = run(b, kernel, first=first, end=end)
    odd = ~np.isfinite(b.v[0])
    assert odd.sum() == (96 if fmt == "q8_0" else 3)
    fine = np.array([~odd[lo:hi].any(0) for lo, hi in zip(first, end)]).reshape(got.shape)
    assert np.array_equal(np.isfinite(got), fine)
    b.v[0][odd] = 0
    want, bar = (x.reshape(got.shape) for x in b.want(first=first, end=end))
    assert (abs(got - want)[fine] <= bar[fine]).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kernel,count", CASES)
@pytest.mark.parametrize("fmt,bad", STORED)
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_a_score_that_is_not_finite_is_reported(device, oracle, cap, bad, kernel, count, dim, fmt):
    ts.say("score, reports", kernel, count, bad, dim, fmt, cap)
    b = ts.Batch(device, oracle, 2, 2, dim, [400], [count], q8=fmt == "q8_0", poison=lambda i, k, v: (ts.put(k, (20, 7), bad), v))
    run(b, kernel, first=np.full(count, 21), end=np.full(count, 330), cap=cap)
    for rows in (slice(None), slice(count - 1, None)):  # all of them, the last
        first = np.full(count, 21)
        first[rows] = 0
        with pytest.raises(_capi.InvalidArgument, match="invalid online attention input"):
            run(b, kernel, first=first, end=np.full(count, 330), cap=cap)
    for bad in (np.inf, np.nan):  # and of a query, where its row sees keys
        b.q[0, 0] = bad
        with pytest.raises(_capi.InvalidArgument, match="invalid online attention input"):
            run(b, kernel, first=np.full(count, 21), end=np.full(count, 330), cap=cap)
        run(b, kernel, first=np.where(np.arange(count), 21, 50), end=np.where(np.arange(count), 330, 50), cap=cap)
