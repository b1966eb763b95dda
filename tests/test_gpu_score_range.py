"""Scored attention over long chunks, whose fp16 parts hold an element to 2^-23 of itself or
2^-39 of its row's largest, over rows of very unequal elements; and the calls that take f32
for every row, which know no such limit."""

import numpy as np
import pytest

import test_gpu_score as ts
from tvara_amd import _capi, attention

pytestmark = pytest.mark.gpu
U, FINE = 2.0 ** -24, 2.0 ** -39
COUNT, N = 170, 200


def run(b, precision, **how):
    """The outputs, by the kernel that the precision stands for."""
    attention.profile_reset()
    attention.profile_enable(True)
    try:
        got = b.run(precision=precision, **how)
        many, few = (attention.profile_read(x)[1] for x in ("score_attention_shared", "score_attention_tiles"))
        assert (many, few) == ((1, 0) if precision == "f32x3" else (0, 1))
    finally:
        attention.profile_enable(False)
    return got


def whole():
    return {"first": np.zeros(COUNT, int), "end": np.full(COUNT, N)}


def of_parts(b):
    """(outputs, bars) of one head's rows over all keys.

    A product of parts is off by 2^-21 of itself (2 x 2^-23, and 2^-22 for low times low), and
    by FINE of each factor's row's largest times the other.  So is a score, whose error doubles in
    its weight; a value is off by FINE of its row's largest, and a weight, times that, by FINE of the
    largest such product.  The f32 sums are the module's (test_gpu_score)."""
    k, v = b.k[0].astype(np.float64), b.v[0].astype(np.float64)
    scale, big = 1 / np.sqrt(b.dim), abs(v).max(1)
    out, bar = np.empty((2, COUNT, b.dim))
    for r in range(COUNT):
        q = b.q[r].astype(np.float64)
        s, size = scale * k @ q, abs(k) @ abs(q)
        off = scale * (((b.dim + 8) * U + 2.0 ** -21) * size + FINE * (abs(q).max() * abs(k).sum(1) + abs(k).max(1) * abs(q).sum()))
        p = np.exp(s - s.max())
        p /= p.sum()
        out[r] = p @ v
        bar[r] = (2 * off.max() + (80 + N / 32) * U + 2.0 ** -20) * (p @ abs(v)) + FINE * (p @ big + 2 * N * (p * big).max())
    return out, bar


@pytest.mark.parametrize("what", ["keys", "queries", "values"])
@pytest.mark.parametrize("power", [0, 12, 24, 30])
@pytest.mark.parametrize("dim", [64, 128])
def test_parts_hold_what_they_are_said_to(device, oracle, dim, power, what):
    ts.say("score, unequal elements, parts", dim, power, what)
    b = unequal(device, oracle, dim, power, what)
    want, bar = of_parts(b)
    assert (abs(run(b, "f32x3", **whole()) - want) <= bar).all()


def unequal(device, oracle, dim, power, what):
    """Column 0 of keys, queries or one value is 2^power times the others; where it would
    drown the scores, the other factor's is 0."""
    def poison(i, k, v):
        if what == "keys":
            k[:, 0] *= 2.0 ** power
        if what == "queries":
            k[:, 0] = 0
        if what == "values":
            v[7, 0] = 2.0 ** power
        return k, v

    b = ts.Batch(device, oracle, 1, 1, dim, [N], [COUNT], poison=poison)
    if what == "keys":
        b.q[:, 0] = 0
    if what == "queries":
        b.q[:, 0] *= 2.0 ** power
    return b


@pytest.mark.parametrize("what", ["keys", "queries", "values"])
@pytest.mark.parametrize("power", [30, 45, 100])
@pytest.mark.parametrize("dim", [64, 128])
def test_f32_has_no_such_limit(device, oracle, dim, power, what):
    ts.say("score, unequal elements, f32", dim, power, what)
    b = unequal(device, oracle, dim, power, what)
    b.agree(run(b, "f32", **whole()), **whole())


@pytest.mark.parametrize("style", list(ts.STYLES))
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
@pytest.mark.parametrize("dim", [64, 128])
def test_f32_over_long_chunks(device, oracle, dim, fmt, style):
    """Chunks of many rows in blocks of sixteen, of two query heads a KV head."""
    ts.say("score, f32, long chunks", dim, fmt, style)
    b = ts.Batch(device, oracle, 4, 2, dim, [331, 170, 200], [170, 170, 1], q8=fmt == "q8_0")
    how = ts.STYLES[style](b)
    b.agree(run(b, "f32", **how), **how)


def test_plans_in_f32(device, oracle):
    ts.say("score, plans in f32")
    b = ts.Batch(device, oracle, 4, 2, 64, [300], [170])
    up = ts.hip.DeviceArray.from_numpy
    q, outs = up(b.q), [ts.hip.DeviceArray(b.q.shape) for _ in range(2)]
    for precision, out in zip(("f32", "f32x3"), outs):
        plan = b.plan(cap=8.0, precision=precision)
        plan.launch(0, q.ptr, out.ptr)
        plan.check()
        b.agree(out.numpy(), cap=8.0)
    assert np.array_equal(outs[0].numpy(), run(b, "f32", cap=8.0)) and not np.array_equal(outs[0].numpy(), outs[1].numpy())
    for precision in ("bf16", "f16", None):
        with pytest.raises(_capi.InvalidArgument, match="f32x3 or f32"):
            b.plan(precision=precision)
        with pytest.raises(_capi.InvalidArgument, match="f32x3 or f32"):
            b.run(precision=precision)
