"""Scored attention over the paged cache on the GPU: capped scores, a bias by
distance, and rows that see ranges of keys of their own, against the formula in
64 bits.

Bars, with u = 2^-24 and each output's own sums.  A score is at most D + 8 rounded
operations on terms of size scale sum_i |q_i k_i|; a cap's tanh adds 8 u cap (its
exponential's argument is off by 3 u of at most 20 where the result still changes, and
then falls in half by each unit), a bias 2 u slope distance.  With e the largest such
error over the row's keys, a probability is off by 2 e + 16 u of itself (its
exponential and the normaliser's), and an output by that and one u a step of 32 keys
and a run that is added, of sum_k p_k |v_k|.  These are worst cases: nothing is to come
near them, and in the 2-norm over many outputs, whose roundings are independent, half
of that is asked for.
"""

import sys

import numpy as np
import pytest

import test_gpu_tree as tt
from tvara_amd import _capi, attention, hip, synth

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def say(*a):
    print(*a, flush=True, file=sys.stderr)


class Batch:
    """Cached sequences and the rows of scored attention over them, in plain arrays too."""

    def __init__(self, device, oracle, heads, kv_heads, dim, lengths, counts, starts=None, tpb=16, q8=False, seed=1,
                 layers=1, poison=None, spare=0):
        self.heads, self.kv_heads, self.dim, self.layers = heads, kv_heads, dim, layers
        self.lengths, self.counts = list(lengths), list(counts)
        self.starts = [n - c for n, c in zip(lengths, counts)] if starts is None else list(starts)
        w = self.w = kv_heads * dim
        blocks = sum(-(-n // tpb) for n in lengths) + 1 + spare
        self.cache = device.PagedCache(layers, kv_heads, dim, tpb, blocks, fmt=device.Q8_0 if q8 else device.F32)
        self.seqs, self.k, self.v = [], [], []
        for i, n in enumerate(lengths):
            k, v = (synth.normal(seed, f"{x}{i}", max(1, n * layers * w))[: n * layers * w].reshape(n, layers * w) for x in "kv")
            if poison:
                k, v = poison(i, k.copy(), v.copy())
            s = self.cache.create_sequence()
            if n:
                self.cache.append_many(s, k, v)
            if q8 and n:
                with np.errstate(all="ignore"):
                    k, v = (oracle.dequantize_q8_0(oracle.quantize_q8_0(x)).reshape(n, layers * w) for x in (k, v))
            self.seqs.append(s)
            self.k.append(k)
            self.v.append(v)
        rows = self.rows = int(sum(counts))
        self.q = 1.5 * synth.normal(seed, "q", max(1, rows * heads * dim))[: rows * heads * dim].reshape(rows, heads * dim)

    def run(self, layer=0, **how):
        return attention.score_batch(self.cache, self.q, self.seqs, self.starts, self.counts, layer, self.heads, 1 << 20, **how)

    def plan(self, **how):
        return attention.ScorePlan(self.cache, self.seqs, self.starts, self.counts, self.heads, 1 << 20, **how)

    def want(self, first=None, end=None, scale=None, cap=0.0, slopes=None, layer=0):
        """(outputs, their bars) in 64 bits."""
        scale = 1 / np.sqrt(self.dim) if scale is None else scale
        out, bar = np.zeros((2, self.rows, self.heads, self.dim))
        cols = slice(layer * self.w, (layer + 1) * self.w)
        g, r = self.heads // self.kv_heads, 0
        for i, c in enumerate(self.counts):
            k, v = (x[i][:, cols].astype(np.float64).reshape(-1, self.kv_heads, self.dim) for x in (self.k, self.v))
            for j in range(c):
                p = self.starts[i] + j
                lo, hi = (0 if first is None else int(first[r])), (p + 1 if end is None else int(end[r]))
                if lo < hi:
                    q = self.q[r].astype(np.float64).reshape(self.heads, 1, self.dim)
                    kk = np.repeat(k[lo:hi], g, 1).transpose(1, 0, 2)
                    vv = np.repeat(v[lo:hi], g, 1).transpose(1, 0, 2)
                    with np.errstate(all="ignore"):
                        s = scale * (q * kk).sum(2)
                        e = (self.dim + 8) * U * scale * (abs(q) * abs(kk)).sum(2)
                        if cap:
                            s = cap * np.tanh(s / cap)
                            e = e + 8 * U * cap
                        if slopes is not None:
                            b = np.asarray(slopes, np.float64)[:, None] * abs(p - np.arange(lo, hi))
                            s, e = s - b, e + 2 * U * abs(b) + U * abs(s)
                        w = np.exp(s - s.max(1, keepdims=True))
                        w /= w.sum(1, keepdims=True)
                        out[r] = (w[:, :, None] * vv).sum(1)
                        rel = 2 * e.max(1) + (16 + (hi - lo) / 32 + 64) * U
                        bar[r] = rel[:, None] * (w[:, :, None] * abs(vv)).sum(1)
                r += 1
        return out.reshape(self.rows, -1), bar.reshape(self.rows, -1)

    def agree(self, got=None, layer=0, **how):
        want, bar = self.want(layer=layer, **how)
        got = np.asarray(self.run(layer=layer, **how) if got is None else got, np.float64)
        assert np.isfinite(got).all()
        off = abs(got - want)
        assert (off <= bar).all(), (float((off / np.maximum(bar, 1e-300)).max()), np.argwhere(off > bar)[:4].tolist())
        assert np.linalg.norm(off) <= 0.5 * np.linalg.norm(bar)
        empty = (bar == 0).all(1)
        assert (got[empty] == 0).all()


def slopes_of(heads):
    return (2.0 ** (-8.0 * np.arange(1, heads + 1) / heads)).astype(np.float32)


STYLES = {
    "plain": lambda b: {},
    "cap": lambda b: {"cap": 6.0},
    "slopes": lambda b: {"slopes": slopes_of(b.heads)},
    "scale, cap and slopes": lambda b: {"scale": 0.3, "cap": 20.0, "slopes": slopes_of(b.heads)},
    "window": lambda b: ranges(b, window=33),
    "window of one": lambda b: ranges(b, window=1),
    "prefix": lambda b: ranges(b, prefix=[n // 2 for n in b.lengths]),
    "documents": lambda b: ranges(b, document=[p // 23 * 23 for s, c in zip(b.starts, b.counts) for p in range(s, s + c)]),
    "any range": lambda b: any_range(b),
}


def ranges(b, **how):
    first, end = attention.visible_ranges(b.starts, b.counts, **how)
    return {"first": first, "end": end}


def any_range(b):
    """Ranges anywhere in the sequence, some of them empty or the wrong way round."""
    r = np.random.default_rng(b.rows)
    first, end = [], []
    for n, c in zip(b.lengths, b.counts):
        lo = r.integers(0, n + 3, c)
        hi = np.minimum(lo + r.integers(-3, n + 1, c), n).clip(0)
        first += lo.tolist()
        end += hi.tolist()
    return {"first": first, "end": end, "cap": 15.0}


@pytest.mark.parametrize("style", list(STYLES))
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("count", [1, 5, 90])
def test_styles(device, oracle, count, dim, fmt, style):
    """Rows of one token, of a few, and of a prompt; lengths around the steps of 32 and 64."""
    say("score", count, dim, fmt, style)
    lengths = [n for n in (1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 95, 128, 200, 331) if n >= count]
    b = Batch(device, oracle, 4, 2, dim, lengths, [count] * len(lengths), q8=fmt == "q8_0", seed=count)
    b.agree(**STYLES[style](b))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (9, 3), (5, 1), (8, 1), (16, 1), (17, 1), (20, 1), (48, 2), (24, 8)])
@pytest.mark.parametrize("count", [1, 4, 37])
def test_groups(device, oracle, heads, kv_heads, count):
    """Query heads that fill a tile's rows, leave some, or go as several blocks."""
    say("score, groups", heads, kv_heads, count)
    b = Batch(device, oracle, heads, kv_heads, 64, [150, 61, 40], [count, min(count, 7), count], seed=heads)
    b.agree(cap=9.0, slopes=slopes_of(heads))


@pytest.mark.parametrize("dim,tpb,fmt", [(32, 16, "f32"), (80, 16, "f32"), (96, 4, "q8_0"), (64, 5, "f32"), (64, 1, "q8_0"), (256, 32, "f32"),
                                         (6, 3, "f32"), (512, 16, "q8_0")])
def test_layouts_without_tiles(device, oracle, dim, tpb, fmt):
    say("score, row by row", dim, tpb, fmt)
    b = Batch(device, oracle, 4, 2, dim, [70, 1, 33], [5, 1, 33], tpb=tpb, q8=fmt == "q8_0")
    b.agree(**STYLES["scale, cap and slopes"](b))
    b.agree(**any_range(b))


@pytest.mark.parametrize("tpb", [16, 64, 256, 1024])
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
def test_blocks(device, oracle, fmt, tpb):
    """Blocks that end inside a step, and blocks of many steps."""
    say("score, blocks", fmt, tpb)
    b = Batch(device, oracle, 8, 2, 128, [1100, 30, 700], [1, 30, 100], tpb=tpb, q8=fmt == "q8_0")
    b.agree(cap=25.0)
    b.agree(**ranges(b, window=300))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
def test_long_contexts_are_cut_and_joined(device, oracle, dim, fmt):
    say("score, long", dim, fmt)
    b = Batch(device, oracle, 8, 2, dim, [20011, 5000, 7], [1, 2, 1], tpb=64, q8=fmt == "q8_0")
    b.agree(cap=30.0, slopes=slopes_of(8) / 64)
    # a range that starts deep inside, and one whose runs a row sees only some of
    b.agree(first=[19000, 10, 4000, 3], end=[20011, 4990, 4001, 7])
    b.agree(first=[19990, 4000, 4990, 9], end=[20000, 4400, 4995, 7])


def test_decoded_rows_and_prompts_in_one_batch(device, oracle):
    say("score, mixed")
    b = Batch(device, oracle, 8, 2, 64, [700, 900, 30, 400, 1], [1, 300, 2, 400, 1], layers=2, starts=[699, 100, 3, 0, 0])
    for layer in (0, 1):
        b.agree(layer=layer, cap=40.0, slopes=slopes_of(8))


def test_a_sequence_listed_twice_and_rows_of_none(device, oracle):
    say("score, twice")
    b = Batch(device, oracle, 4, 2, 64, [90, 50], [3, 0])
    b.seqs, b.starts, b.counts = [b.seqs[0], b.seqs[0], b.seqs[1]], [5, 60, 50], [2, 1, 0]
    b.lengths, b.k, b.v = [90, 90, 50], [b.k[0], b.k[0], b.k[1]], [b.v[0], b.v[0], b.v[1]]
    b.agree(cap=5.0)
    none = attention.ScorePlan(b.cache, [b.seqs[0]], [3], [0], 4, 1 << 20)
    none.launch(0, None, None)
    none.check()


@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("count", [1, 3, 80])
@pytest.mark.parametrize("bad", [np.inf, np.nan, 3.4e38])
def test_what_a_row_does_not_see_never_reaches_it(device, oracle, bad, count, dim, fmt):
    """Keys and values behind, before and between the visible ones, whatever they hold."""
    if fmt == "q8_0" and bad == 3.4e38:
        bad = 1e30  # (its scale is infinite)
    say("score, unseen", bad, count, dim, fmt)
    n = 200
    hidden = [0, 3, 40, 41, 77, n - 1]

    def poison(i, k, v):
        k[hidden], v[hidden] = bad, bad
        return k, v

    b = Batch(device, oracle, 4, 2, dim, [n], [count], q8=fmt == "q8_0", poison=poison)
    gaps = [(4, 40), (42, 77), (78, n - 1), (1, 3), (5, 5)]
    first, end = (np.array([gaps[j % 5][e] for j in range(count)]) for e in (0, 1))
    for x in (b.k, b.v):
        x[0] = np.nan_to_num(x[0], nan=0, posinf=0, neginf=0)  # (the 64-bit form multiplies ranges only)
    b.agree(first=first, end=end)


@pytest.mark.parametrize("count", [1, 3, 80])
@pytest.mark.parametrize("dim", [64, 96])
def test_what_is_not_finite_shows(device, oracle, count, dim):
    """A value reaches its column of the rows that see it and no other; a score is reported."""
    say("score, not finite", count, dim)
    b = Batch(device, oracle, 4, 2, dim, [120], [count], poison=lambda i, k, v: (k, put(v, (20, dim + 7), np.inf)))
    first = np.where(np.arange(count) % 2, 21, 0)
    got = b.run(first=first, end=np.full(count, 40)).reshape(count, 4, dim)
    fine = np.ones(got.shape, bool)
    fine[::2, 2:, 7] = False
    assert np.array_equal(np.isfinite(got), fine)
    b.v[0][20, dim + 7] = 0
    want, bar = b.want(first=first, end=np.full(count, 40))
    off = abs(got.reshape(count, -1) - want)
    assert (off[fine.reshape(count, -1)] <= bar[fine.reshape(count, -1)]).all()
    for cap in (0.0, 5.0):
        b = Batch(device, oracle, 4, 2, dim, [120], [count], poison=lambda i, k, v: (put(k, (20, 7), np.inf), v))
        b.run(first=np.full(count, 21), end=np.full(count, 40), cap=cap)
        with pytest.raises(_capi.InvalidArgument):
            b.run(first=first, end=np.full(count, 40), cap=cap)


def put(x, at, value):
    x[at] = value
    return x


@pytest.mark.parametrize("count", [1, 66])
@pytest.mark.parametrize("dim", [64, 128, 32])
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
def test_small_weights_add_up(device, oracle, fmt, dim, count):
    """Beside the largest weight the others are each less than half an ulp of the sums,
    and together many: one key 19 above 32,767 others, values all of one sign."""
    say("score, small weights", fmt, dim, count)
    n = 32768

    def poison(i, k, v):
        u = np.zeros(k.shape[1], np.float32)
        u[0] = 19 * np.sqrt(dim)
        k[:] = 0
        k[5] = u
        v[:] = 1
        v[5] = 0.5
        return k, v

    b = Batch(device, oracle, 1, 1, dim, [n], [count], q8=fmt == "q8_0", tpb=64, poison=poison)
    b.q[:] = 0
    b.q[:, 0] = 1
    whole = {"first": np.zeros(count, int), "end": np.full(count, n)}
    got = b.run(**whole).astype(np.float64)
    want, _ = b.want(**{k: v[:1] for k, v in whole.items()}) if count == 1 else (None, None)
    s = float(b.k[0][5, 0]) / np.sqrt(dim)
    exact = (0.5 + (n - 1) * np.exp(-s)) / (1 + (n - 1) * np.exp(-s)) if fmt == "f32" else None
    if want is not None:
        exact = want[0, 0] if exact is None else exact
    if exact is None:
        v = b.v[0][:, 0].astype(np.float64)
        w = np.exp(b.k[0][:, 0] / np.sqrt(dim) - s)
        exact = (w * v).sum() / w.sum()
    # A run is of 4 steps or 64 keys here, so a sum has up to 4 additions in a run, 3 where
    # waves join, twice, and 2 u in a compensated merge; a division is u more; what is
    # left (of e^-s, 2 u s) is of the small part.  Together less than 16 u.
    assert np.max(abs(got - exact)) <= 1e-6, (float(got[0, 0]), exact)


def test_far_positions(device, oracle):
    """Distances that f32 holds as whole numbers, and a bias that leaves the last keys only."""
    say("score, far")
    b = Batch(device, oracle, 4, 2, 64, [70001], [2], tpb=256)
    b.agree(slopes=[0.0, 1e-4, 0.5, 20.0])


@pytest.mark.parametrize("count", [1, 100])
def test_captured_launches(device, oracle, count):
    """A graph of two layers' launches, replayed with eager work between."""
    say("score, captured", count)
    b = Batch(device, oracle, 8, 2, 64, [3000, 200], [count, count], layers=2)
    stream = hip.Stream()
    hip.synchronize()
    b.cache.set_stream(stream.h)
    up = hip.DeviceArray.from_numpy
    plan = b.plan(cap=30.0)
    q, outs = up(b.q), [hip.DeviceArray(b.q.shape) for _ in range(2)]

    def both():
        for layer, out in enumerate(outs):
            plan.launch(layer, q.ptr, out.ptr, stream=stream.h)

    both()
    plan.check()
    eager = [o.numpy() for o in outs]
    graph = tt.Graph(stream.h, both)
    for _ in range(3):
        for o in outs:
            o.zero()
        hip.synchronize()
        graph.replay()
        plan.check()
        for o, e in zip(outs, eager):
            assert np.array_equal(o.numpy(), e)
    for layer, e in enumerate(eager):
        b.agree(e, layer=layer, cap=30.0)
    del graph
    hip.synchronize()
    b.cache.set_stream(None)


def test_other_streams_and_stale_plans(device, oracle):
    say("score, streams")
    b = Batch(device, oracle, 4, 2, 64, [300], [4], spare=2)
    up = hip.DeviceArray.from_numpy
    q, out = up(b.q), hip.DeviceArray(b.q.shape)
    stream = hip.Stream()
    plan = b.plan(cap=8.0)
    plan.launch(0, q.ptr, out.ptr, stream=stream.h)
    plan.check()
    b.agree(out.numpy(), cap=8.0)
    b.cache.append(b.seqs[0], np.zeros(b.w), np.zeros(b.w))
    with pytest.raises(_capi.InvalidArgument, match="stale"):
        plan.launch(0, q.ptr, out.ptr)


def test_refusals(device, oracle):
    say("score, refusals")
    b = Batch(device, oracle, 4, 2, 64, [40, 30], [2, 1])
    c, s = b.cache, b.seqs
    up = hip.DeviceArray.from_numpy(np.zeros(8 * 256, np.float32))
    bad = _capi.InvalidArgument

    def make(seqs=s, starts=(38, 29), counts=(2, 1), heads=4, context=1 << 20, **how):
        return attention.ScorePlan(c, seqs, starts, counts, heads, context, **how)

    for how in ({"heads": 3}, {"heads": 0}, {"context": 0}, {"context": 39}, {"starts": (39, 29)}, {"starts": (41, 29), "counts": (0, 1)},
                {"starts": (38,)}, {"counts": (2, -1)}, {"starts": (0.5, 1)}, {"scale": -1.0}, {"scale": np.nan}, {"scale": np.inf},
                {"cap": -1.0}, {"cap": np.nan}, {"cap": np.inf}, {"slopes": [1.0]}, {"slopes": [1.0, 1.0, np.nan, 1.0]},
                {"first": [0, 0]}, {"end": [39, 41, 30]}, {"end": [39, 40, 31]}, {"first": [-1, 0, 0]}, {"seqs": []}):
        with pytest.raises(bad):
            make(**how)
    with pytest.raises(_capi.NativeError):
        make(seqs=[s[0], 999])
    plan = make()
    for call in (lambda: plan.launch(1, up.ptr, up.ptr), lambda: plan.launch(0, None, up.ptr), lambda: plan.launch(0, up.ptr, None),
                 lambda: plan.launch(0, up.ptr + 4, up.ptr), lambda: plan.launch(1 << 40, up.ptr, up.ptr)):
        with pytest.raises(bad):
            call()
    plan.launch(0, up.ptr, up.ptr + 4 * 1024)
    plan.check()
    plan.close()
    for x in (b.k, b.v):
        assert all(np.isfinite(y).all() for y in x)
    b.agree(cap=3.0)


def test_more_rows_than_a_launch_holds(device, oracle):
    say("score, too many rows")
    b = Batch(device, oracle, 1, 1, 16, [20], [1])
    for rows in (1 << 24, 1 << 40):
        with pytest.raises(_capi.InvalidArgument, match="too large"):
            attention.ScorePlan(b.cache, b.seqs, [0], [rows], 1, 1 << 20)
    b.agree()
