"""Scored attention whose workgroups walk whole contexts alone: long sums of small parts
behind a large one, and the sums of many rows on their way through memory.

Sequences are listed so often that every CU has its workgroups and none of their keys are cut
into runs by the batch's size: 256 blocks of many rows, or of few in f32, 768 of few in Q8_0,
4,096 (row, head) pairs of the row kernel.
"""

import numpy as np
import pytest

import test_gpu_score as ts
from tvara_amd import attention

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
KERNELS = {"many": "score_attention_shared", "few": "score_attention_tiles"}


def listed(b, times, kernel, **how):
    """The outputs of b's rows, listed `times` times with the same queries, which are to
    be equal bit for bit; `kernel` is what has to have run."""
    given = {k: np.tile(v, times) if k in ("first", "end") else v for k, v in how.items()}
    attention.profile_reset()
    attention.profile_enable(True)
    try:
        got = attention.score_batch(b.cache, np.tile(b.q, (times, 1)), b.seqs * times, b.starts * times, b.counts * times, 0, b.heads,
                                    1 << 20, **given)
        launches = {k: attention.profile_read(name)[1] for k, name in KERNELS.items()}
        assert launches == {k: int(k == kernel) for k in KERNELS}, launches
    finally:
        attention.profile_enable(False)
    got = got.reshape(times, *b.q.shape)
    assert np.array_equal(got, np.broadcast_to(got[:1], got.shape), equal_nan=True)
    return got[0]


@pytest.mark.parametrize("kernel,dim,fmt,count,times,heads,added", [
    # added: additions in a row to sums that hold the large part
    ("many", 64, "f32", 170, 256, 1, 128 + 8), ("many", 128, "f32", 170, 256, 1, 128 + 16),
    ("many", 64, "q8_0", 170, 256, 1, 128 + 8), ("many", 128, "q8_0", 170, 256, 1, 128 + 16),
    ("few", 64, "f32", 1, 256, 1, 64 + 3), ("few", 128, "f32", 1, 256, 1, 64 + 3),
    ("few", 64, "q8_0", 1, 768, 1, 64 + 3), ("few", 128, "q8_0", 1, 768, 1, 64 + 3),
    ("row", 32, "f32", 1, 256, 16, 64), ("row", 96, "q8_0", 1, 256, 16, 64), ("row", 256, "f32", 1, 256, 16, 64),
])
def test_small_parts_add_up(device, oracle, kernel, dim, fmt, count, times, heads, added):
    """One key 21 above 65,535 others, values of one sign: a step's part of the others, 32 or 64
    times e^-21, is less than half an ulp of the large key's, and all of them 5e-5 of it.

    A sum is off by at most half an ulp, u of it, for each of the additions that it takes in
    a row; all but these are compensated.  Beside that go 16 u for the products, the normaliser
    and the division, and for e^-21, which is off by 2^-18 of 5e-5."""
    ts.say("score, small parts", kernel, dim, fmt)
    n = 65536

    def poison(i, k, v):
        k[:] = 0
        k[5, 0] = 21 * np.sqrt(dim)
        return k, 1 + 0.25 * np.tanh(v)

    b = ts.Batch(device, oracle, heads, 1, dim, [n], [count], tpb=64, q8=fmt == "q8_0", poison=poison)
    b.q[:] = 0
    b.q.reshape(-1, dim)[:, 0] = 1
    got = listed(b, times, kernel, first=np.zeros(count, int), end=np.full(count, n)).reshape(-1, dim).astype(np.float64)
    s = b.k[0][:, 0].astype(np.float64) / np.sqrt(dim)
    w = np.exp(s - s[5])
    want = w @ b.v[0].astype(np.float64) / w.sum()
    assert w.sum() - 1 > 4.5e-5
    assert (abs(got - want) <= (added + 16) * U * want).all(), float((abs(got - want) / want).max())


def rising(i, k, v):
    """Scores that grow along the sequence, so that maxima change after sums were put down."""
    return k * np.linspace(0.2, 3, len(k), dtype=np.float32)[:, None], v


@pytest.mark.parametrize("style", ["plain", "rising", "falling", "ranges", "cap and slopes"])
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
@pytest.mark.parametrize("dim", [64, 128])
def test_sums_of_many_rows_through_memory(device, oracle, dim, fmt, style):
    """Contexts of two and a bit times the steps after which they go there (4,096 keys of 128
    columns, 8,192 of 64)."""
    ts.say("score, sums through memory", dim, fmt, style)
    n, count = {64: 16500, 128: 9001}[dim], 170
    poison = {"rising": rising, "falling": lambda i, k, v: tuple(x[::-1] for x in rising(i, k[::-1], v[::-1]))}.get(style)
    b = ts.Batch(device, oracle, 1, 1, dim, [n], [count], tpb=256, q8=fmt == "q8_0", poison=poison)
    how = {"first": np.zeros(count, int), "end": np.full(count, n)}
    if style == "ranges":  # keys before, behind and across the borders, and none
        at = {64: 8192, 128: 4096}[dim]
        some = [(0, n), (at, n), (at + 1, at + 40), (5, at), (2 * at, n), (0, 0), (n - 1, n), (at - 3, 2 * at + 3), (n, 3), (7, 8)]
        how = {e: np.array([some[r % len(some)][i] for r in range(count)]) for i, e in enumerate(("first", "end"))}
    if style == "cap and slopes":
        how.update(cap=30.0, slopes=[2.0 ** -10])
    b.agree(listed(b, 256, "many", **how), **how)


@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_not_finite_after_sums_through_memory(device, oracle, dim):
    """A value shows in its column of the rows that see it, whichever part of the context has it."""
    ts.say("score, not finite, through memory", dim)
    n, count, at = {64: 16500, 128: 9001}[dim], 170, {64: 8192, 128: 4096}[dim]
    holes = [(9, 3), (at + 70, 5), (n - 2, dim - 1)]

    def poison(i, k, v):
        for where in holes:
            v[where] = np.inf
        return k, v

    b = ts.Batch(device, oracle, 1, 1, dim, [n], [count], tpb=256, poison=poison)
    first = np.where(np.arange(count) % 2, at + 71, 0)
    end = np.where(np.arange(count) % 3, n, n - 2)
    got = listed(b, 256, "many", first=first, end=end)
    fine = np.ones(got.shape, bool)
    for key, column in holes:
        fine[(first <= key) & (key < end), column] = False
        b.v[0][key, column] = 0
    assert np.array_equal(np.isfinite(got), fine)
    want, bar = b.want(first=first, end=end)
    assert (abs(got - want)[fine] <= bar[fine]).all()


def test_sums_through_memory_in_runs(device, oracle):
    """Contexts that are cut into runs which are still that long."""
    ts.say("score, runs through memory")
    n, count, times = 30000, 170, 100
    b = ts.Batch(device, oracle, 1, 1, 128, [n], [count], tpb=256, poison=rising)
    how = {"first": np.arange(count) * 150, "end": np.full(count, n)}
    b.agree(listed(b, times, "many", **how), **how)
