"""Sampling on the GPU against its definition in 64 bits: temperature, top-k, top-p and
min-p from given random numbers.

Tokens are whole numbers and equal.  The kernel's masses are off by at most 2^-45 of the
largest weight for each token and 1e-14 of each weight, numpy's by 1e-15: over 300,000
tokens 1e-8 of the largest weight at the very worst and 1e-11 as independent roundings
go.  A random number, a top-p or a min-p nearer to a border than that may fall on either
side; the reference says how near it comes, and inputs here stay away by 1e-10 or are
exact in both (ties, powers of two).  A probability is the weight over the mass, rounded
to f32: 2^-24 and those 1e-10 beside it.
"""

import sys

import numpy as np
import pytest

import test_gpu_tree as tt
from tvara_amd import _capi, hip
from tvara_amd.sampling import SamplePlan, sample_batch

pytestmark = pytest.mark.gpu
NONE = 0xFFFFFFFF


def say(*a):
    print(*a, flush=True, file=sys.stderr)


def draw(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """(token, probability) of one row."""
    t, p, m, u = (float(np.float32(y)) for y in (t, p, m, u))
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if x.max() == -np.inf:
        return NONE, 0.0
    order = np.argsort(-x, kind="stable")
    if t == 0 or k == 1 or p == 0:
        return int(order[0]), 1.0
    with np.errstate(all="ignore"):
        w = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / t))
    order = order[: k or None]
    mass = np.cumsum(w[order])
    keep = order[(mass - w[order] < p * mass[-1]) & (w[order] >= m)]
    kept = np.zeros_like(w)
    kept[keep] = w[keep]
    upto = np.cumsum(kept)
    token = int(np.searchsorted(upto, u * upto[-1], side="right"))
    return token, kept[token] / upto[-1]


def agree(x, u, t=1.0, k=0, p=1.0, m=0.0):
    x, u = np.atleast_2d(np.asarray(x, np.float32)), np.asarray(u, np.float32)
    got, chance = sample_batch(x, u, t, k, p, m)
    each = [np.broadcast_to(np.asarray(y), u.shape) for y in (t, k, p, m)]
    for i, row in enumerate(x):
        token, probability = draw(row, u[i], *(y[i] for y in each))
        assert got[i] == token, (i, int(got[i]), token, float(chance[i]), probability)
        assert abs(chance[i] - probability) <= (2.0 ** -24 + 1e-9) * probability, (i, chance[i], probability)


def logits(rng, n, vocab, sigma=2.0, likely=16.0, bf16=True):
    x = sigma * rng.normal(size=(n, vocab))
    for row in x:
        at = rng.integers(0, vocab, 24)
        row[at] += likely * rng.random() * rng.random(24)
    x = x.astype(np.float32)
    return (x.view(np.uint32) & 0xFFFF0000).view(np.float32) if bf16 else x


PARAMS = [{}, {"t": 0.7}, {"t": 1.5}, {"k": 1}, {"k": 5}, {"k": 50}, {"k": 2000}, {"p": 0.9}, {"p": 0.5, "t": 0.8}, {"p": 0.01}, {"p": 0.999},
          {"m": 0.05}, {"m": 1.0}, {"m": 1e-4, "t": 1.3}, {"k": 50, "p": 0.9}, {"k": 3, "p": 0.3, "m": 0.1}, {"k": 1500, "p": 0.95, "t": 1.2},
          {"k": 40, "m": 0.02, "t": 0.6}, {"p": 0.97, "m": 0.01}, {"t": 0.0}, {"t": 1e-3}, {"t": 50.0}, {"t": 50.0, "p": 0.6}, {"p": 0.0}]


@pytest.mark.parametrize("what", PARAMS, ids=lambda w: " ".join(f"{k}={v}" for k, v in w.items()) or "plain")
@pytest.mark.parametrize("vocab", [1, 2, 7, 255, 256, 257, 1024, 5000, 32000])
def test_parameters(vocab, what):
    say("sample", vocab, what)
    rng = np.random.default_rng(vocab)
    agree(logits(rng, 12, vocab), rng.random(12), **what)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("sigma,likely", [(0.0, 0.0), (0.3, 0.0), (2.5, 0.0), (2.0, 30.0), (8.0, 0.0)])
@pytest.mark.parametrize("vocab", [128256, 300001])
def test_large_vocabularies(vocab, sigma, likely, bf16):
    """Flat, ordinary and sharp rows; with one value alone every logit is a tie."""
    say("sample, large", vocab, sigma, likely, bf16)
    rng = np.random.default_rng(int(10 * sigma) + vocab)
    x = logits(rng, 4, vocab, sigma, likely, bf16)
    for what in ({}, {"p": 0.9}, {"k": 40}, {"k": 9000}, {"k": 9000, "p": 0.8}, {"m": 0.01}, {"t": 0.0}):
        agree(x, rng.random(4), **what)


@pytest.mark.parametrize("vocab", [300, 6000, 20000])
def test_ties(vocab):
    """Equal logits are taken by index: at top-k's border, top-p's, and the maximum."""
    say("sample, ties", vocab)
    n = 16
    rng = np.random.default_rng(vocab)
    u = (rng.integers(0, 1 << 12, n) + 0.5) / (1 << 12)
    same = np.zeros((n, vocab), np.float32)
    for k in (0, 1, 2, 255, 256, vocab // 2, vocab - 1, vocab, vocab + 5):
        agree(same, u, k=k)
    for p in (0.25, 0.5, 1.0, 0.75):
        agree(same, u, p=p)
        agree(same, u, k=vocab // 2, p=p)
    # two levels: weights 1 and 2^-3 exactly, at T = 3 ln 2 / 3
    two = np.where(rng.random((n, vocab)) < 0.02, 3.0, 0.0).astype(np.float32)
    for k in (0, 3, int(two[0].sum() / 3), int(two[0].sum() / 3) + 7, vocab // 2):
        agree(two, u, k=k, t=1.4)
        agree(two, u, k=k, t=1.4, p=0.3)
        agree(two, u, k=k, t=1.4, p=0.8, m=0.5)
    agree(-two, u, t=0.0)
    agree(two, u, t=0.0)
    zeros = np.where(rng.random((n, vocab)) < 0.5, np.float32(0.0), np.float32(-0.0))
    agree(zeros, u, k=vocab // 3)
    agree(zeros, u, t=0.0)


def test_masked_and_extreme_logits():
    say("sample, extremes")
    rng = np.random.default_rng(5)
    n, vocab, low = 8, 3000, float(np.finfo(np.float32).min)
    u = rng.random(n)
    for fill in (-np.inf, low):
        x = np.full((n, vocab), fill, np.float32)
        some = rng.integers(0, vocab, (n, 9))
        np.put_along_axis(x, some, rng.normal(size=(n, 9)).astype(np.float32), 1)
        for what in ({}, {"k": 4}, {"k": 500}, {"p": 0.8}, {"m": 0.3}, {"t": 0.0}, {"k": 500, "p": 0.8}):
            agree(x, u, **what)
    agree(np.full((n, vocab), low), u)
    agree(np.full((n, vocab), low), u, k=17, p=0.5)
    # one infinite logit, and several
    x = rng.normal(size=(n, vocab)).astype(np.float32)
    x[:, 70] = np.inf
    for what in ({}, {"k": 4}, {"p": 0.8}, {"m": 0.3}, {"t": 0.0}):
        agree(x, u, **what)
    x[:, 1700] = np.inf
    for what in ({}, {"k": 4}, {"p": 0.8}, {"t": 0.0}):
        agree(x, u, **what)
    # the whole range of f32
    wide = (rng.normal(size=(n, vocab)) * 1e38).astype(np.float32)
    for what in ({}, {"k": 4}, {"p": 0.8}, {"t": 3e38}, {"t": 3e38, "k": 100, "p": 0.7}):
        agree(wide, u, **what)
    for t in (1e-30, 1e-45, 1e30):
        agree(x[:, :60], u, t=t)
        agree(x[:, :60], u, t=t, p=0.6, k=11)
    # random numbers at the ends
    y = logits(rng, 4, vocab)
    ends = [0.0, np.nextafter(np.float32(1), np.float32(0)), 2.0 ** -30, 0.5]
    for what in ({}, {"k": 30}, {"p": 0.9}, {"m": 0.1}):
        agree(y, ends, **what)


def test_rows_of_their_own():
    """Parameters by row, a row's stride beyond its vocabulary, more room than rows."""
    say("sample, by row")
    rng = np.random.default_rng(9)
    n, vocab = 40, 4321
    x, u = logits(rng, n, vocab), rng.random(n).astype(np.float32)
    t, p, m = (rng.choice(c, n).astype(np.float32) for c in ([0.0, 0.5, 1.0, 1.7], [1.0, 0.9, 0.3], [0.0, 0.0, 0.1]))
    k = rng.choice([0, 1, 20, 1000], n).astype(np.int32)
    agree(x, u, t, k, p, m)
    want, chance = sample_batch(x, u, t, k, p, m)
    up = hip.DeviceArray.from_numpy
    for stride in (vocab + 3, vocab + 7):  # (a multiple of 4, and not)
        wide = np.full((n, stride), 100.0, np.float32)
        wide[:, :vocab] = x
        d = [up(y) for y in (wide, u, t, k, p, m)]
        tokens, chances = up(np.full(n + 2, 7, np.uint32)), hip.DeviceArray((n,))
        plan = SamplePlan(n + 10, vocab)
        plan.launch(d[0].ptr, d[1].ptr, tokens.ptr, chances.ptr, d[2].ptr, d[3].ptr, d[4].ptr, d[5].ptr, rows=n, logits_stride=stride)
        plan.check()
        assert np.array_equal(tokens.numpy(), [*want, 7, 7]) and np.array_equal(chances.numpy(), chance)
        plan.launch(None, None, None, rows=0)
        plan.check()
    # the same rows in another batch
    again, _ = sample_batch(x[3:9], u[3:9], t[3:9], k[3:9], p[3:9], m[3:9])
    assert np.array_equal(again, want[3:9])


def test_frequencies():
    """Drawn by evenly spaced numbers, every token comes as often as its probability says."""
    say("sample, frequencies")
    n = 4096
    x = np.log(np.array([0.5, 0.25, 0.125, 0.0625, 0.0625])).astype(np.float32)
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    tokens, _ = sample_batch(np.broadcast_to(x, (n, 5)), u)
    # (logs of powers of two in f32 are off by 2^-24: less than half a step of u)
    assert np.bincount(tokens).tolist() == [2048, 1024, 512, 256, 256]
    tokens, _ = sample_batch(np.broadcast_to(x, (n, 5)), u, top_p=0.7)
    counts = np.bincount(tokens)
    assert counts.size == 2 and abs(counts[0] - n * 2 / 3) <= 1


@pytest.mark.parametrize("vocab", [500, 40000])
def test_what_cannot_be_drawn_is_reported(vocab):
    say("sample, reports", vocab)
    rng = np.random.default_rng(1)
    x, u = logits(rng, 5, vocab), rng.random(5).astype(np.float32)
    good, _ = sample_batch(x, u)
    up = hip.DeviceArray.from_numpy
    plan = SamplePlan(5, vocab)

    def run(x=x, u=u, t=None, k=None, p=None, m=None):
        d = [None if y is None else up(np.asarray(y)) for y in (x, u, t, k, p, m)]
        tokens, chances = hip.DeviceArray((5,), np.uint32), hip.DeviceArray((5,))
        ptr = [y and y.ptr for y in d]
        plan.launch(ptr[0], ptr[1], tokens.ptr, chances.ptr, *ptr[2:])
        try:
            plan.check()
            message = ""
        except _capi.InvalidArgument as e:
            message = str(e)
        return tokens.numpy(), chances.numpy(), message

    one = np.ones(5, np.float32)
    bad = x.copy()
    bad[1, 7] = np.nan
    bad[3] = -np.inf
    bad[4] = np.nan
    tokens, chances, message = run(bad)
    assert "invalid logits" in message
    assert tokens[3] == tokens[4] == NONE and chances[3] == chances[4] == 0 and tokens[0] == good[0] and tokens[2] == good[2]
    assert tokens[1] == draw(bad[1], u[1])[0]
    for what, value in (("u", 1.0), ("u", -0.1), ("u", np.nan), ("t", -1.0), ("t", np.inf), ("t", np.nan), ("p", 1.5), ("p", -0.1),
                        ("p", np.nan), ("m", -0.5), ("m", 1.1), ("m", np.nan), ("k", -1)):
        given = {"u": u, "t": one, "p": one, "m": 0 * one, "k": np.zeros(5, np.int32)}[what].copy()
        given[2] = value
        tokens, chances, message = run(**{what: given})
        assert "invalid sampling parameters" in message, (what, value)
        assert tokens[2] == NONE and chances[2] == 0
        assert np.array_equal(np.delete(tokens, 2), np.delete(good, 2))
    assert run()[2] == ""


def test_captured_and_on_another_stream():
    say("sample, captured")
    rng = np.random.default_rng(2)
    x, u = logits(rng, 6, 70000), rng.random(6).astype(np.float32)
    up = hip.DeviceArray.from_numpy
    d, du, p = up(x), up(u), up(np.full(6, 0.9, np.float32))
    tokens, chances = hip.DeviceArray((6,), np.uint32), hip.DeviceArray((6,))
    plan, stream = SamplePlan(6, 70000), hip.Stream()
    hip.synchronize()

    def launch():
        plan.launch(d.ptr, du.ptr, tokens.ptr, chances.ptr, top_p_ptr=p.ptr, stream=stream.h)

    launch()
    plan.check()
    want = tokens.numpy()
    assert [int(t) for t in want] == [draw(x[i], u[i], p=0.9)[0] for i in range(6)]
    graph = tt.Graph(stream.h, launch)
    for _ in range(3):
        tokens.zero()
        chances.zero()
        hip.synchronize()
        graph.replay()
        plan.check()
        assert np.array_equal(tokens.numpy(), want) and (chances.numpy() > 0).all()
    del graph


def test_refusals():
    say("sample, refusals")
    bad = _capi.InvalidArgument
    for rows, vocab in ((0, 5), (5, 0), (1, 1 << 31), (1 << 31, 1), (1 << 20, 1 << 20)):
        with pytest.raises(bad):
            SamplePlan(rows, vocab)
    up = hip.DeviceArray.from_numpy
    d = up(np.zeros(64, np.float32))
    plan = SamplePlan(2, 8)
    for args, how in (((None, d.ptr, d.ptr), {}), ((d.ptr, None, d.ptr), {}), ((d.ptr, d.ptr, None), {}), ((d.ptr + 4, d.ptr, d.ptr), {}),
                      ((d.ptr, d.ptr, d.ptr), {"rows": 3}), ((d.ptr, d.ptr, d.ptr), {"logits_stride": 7}),
                      ((d.ptr, d.ptr, d.ptr), {"top_p_ptr": d.ptr + 8})):
        with pytest.raises(bad):
            plan.launch(*args, **how)
    x = np.zeros((2, 8))
    for how in ({"top_k": -1}, {"top_k": 0.5}, {"top_k": 1 << 40}, {"top_p": [1.0]}, {"temperature": [1.0, 1.0, 1.0]}):
        with pytest.raises(bad):
            sample_batch(x, [0.1, 0.2], **how)
    with pytest.raises(bad):
        sample_batch(x, [0.1])
    with pytest.raises(bad):
        sample_batch(x[0], [0.1])
    assert sample_batch(np.zeros((0, 8)), [])[0].size == 0


def test_rows_that_pass_the_address_space_are_refused():
    say("sample, strides without end")
    d, plan = hip.DeviceArray.from_numpy(np.zeros(64, np.float32)), SamplePlan(4, 8)
    for stride in (1 << 62, 1 << 58, (1 << 64) - 4):
        with pytest.raises(_capi.InvalidArgument, match="overlap"):
            plan.launch(d.ptr, d.ptr, d.ptr, logits_stride=stride)
    plan.check()
