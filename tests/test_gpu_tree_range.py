"""Tree attention over the whole range of its inputs: weights far below a row's
largest, values far from one, values that f32x3's fp16 parts do not hold.  The bars are test_gpu_tree's unless a test derives its own."""

import numpy as np
import pytest

import test_gpu_tree as tt
from tvara_amd import _capi, attention, synth

pytestmark = pytest.mark.gpu
ROWS = ["16", "32", "128"]  # that a workgroup of f32x3 may have


class Sink:
    """One sequence under 256 trees of a node: its first key's score is `gap`, the
    others' are N(0,1).  256 trees of two KV heads give every CU its workgroups, so
    each walks the whole context alone."""

    TREES, KV, GROUP, CHECKED = 256, 2, 2, 24

    def __init__(self, device, oracle, dim, n, gap, q8, sink_value=1.0):
        w, self.dim, self.n = self.KV * dim, dim, n
        u = synth.normal(dim, "u", w).reshape(self.KV, dim).astype(np.float64)
        u /= np.linalg.norm(u, axis=1, keepdims=True)
        k, v, q, tk, tv = (synth.normal(n, x, rows * c).reshape(rows, -1, dim).astype(np.float64) for x, rows, c in (
            ("k", n, w), ("v", n, w), ("q", self.TREES, self.GROUP * w), ("tk", self.TREES, w), ("tv", self.TREES, w)))
        along = np.repeat(u, self.GROUP, 0)
        q += (np.sqrt(dim) - (q * along).sum(2, keepdims=True)) * along  # sqrt(dim) along u
        for x in (k, tk):
            x -= (x * u).sum(2, keepdims=True) * u
        k[0], v[0] = gap * u, sink_value * v[0]
        k, v, tk, tv = (np.ascontiguousarray(x.reshape(-1, w), np.float32) for x in (k, v, tk, tv))
        self.q = np.ascontiguousarray(q.reshape(self.TREES, -1), np.float32)
        self.cache = device.PagedCache(1, self.KV, dim, 64, n // 64 + 1, fmt=device.Q8_0 if q8 else device.F32)
        self.seq = self.cache.create_sequence()
        self.cache.append_many(self.seq, k, v)
        if q8:
            k, v = (oracle.dequantize_q8_0(oracle.quantize_q8_0(x)).reshape(n, w) for x in (k, v))
        self.k, self.v, self.tk, self.tv = k, v, tk, tv

    def run(self, precision):
        n = self.TREES
        got = attention.tree_batch(self.cache, self.q, [self.seq] * n, [1] * n, [-1] * n, self.tk, self.tv, 0,
                                   self.KV * self.GROUP, 1 << 20, precision=precision)
        return got[: self.CHECKED].reshape(self.CHECKED, -1, self.dim).astype(np.float64)

    def want(self):
        out = np.empty((self.CHECKED, self.KV * self.GROUP, self.dim))
        for h in range(out.shape[1]):
            cols = slice(h // self.GROUP * self.dim, (h // self.GROUP + 1) * self.dim)
            x = self.q.reshape(self.TREES, -1, self.dim)[: self.CHECKED, h].astype(np.float64)
            tk, tv = (y[: self.CHECKED, cols].astype(np.float64) for y in (self.tk, self.tv))
            s = np.concatenate([x @ self.k[:, cols].astype(np.float64).T, (x * tk).sum(1, keepdims=True)], 1) / np.sqrt(self.dim)
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            out[:, h] = p[:, :-1] @ self.v[:, cols].astype(np.float64) + p[:, -1:] * tv
        return out


@pytest.mark.parametrize("gap", [12, 18, 19.5, 21])
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
@pytest.mark.parametrize("dim", [64, 128])
def test_small_weights_add_up(device, oracle, dim, fmt, gap):
    """Beside the largest weight each step's others may be less than half an ulp of the
    normaliser, and together many."""
    tt.say("tree, one key far above, f32", dim, fmt, gap)
    b = Sink(device, oracle, dim, 32768, gap, fmt == "q8_0")
    tt.agree(b.run("f32"), b.want(), "f32")


@pytest.mark.parametrize("gap", [12, 16, 18, 19.5])
@pytest.mark.parametrize("n", [4096, 32768])
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
@pytest.mark.parametrize("dim", [64, 128])
def test_one_key_far_above_many(device, oracle, monkeypatch, dim, fmt, n, gap):
    tt.say("tree, one key far above", dim, fmt, n, gap)
    b = Sink(device, oracle, dim, n, gap, fmt == "q8_0")
    want = b.want()
    for rows in ROWS:
        monkeypatch.setenv("TVARA_TREE_ROWS", rows)
        tt.agree(b.run("f32x3"), want, "f32x3")


@pytest.mark.parametrize("gap", [12, 18])
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
@pytest.mark.parametrize("dim", [64, 128])
def test_one_key_far_above_without_a_value(device, oracle, monkeypatch, dim, fmt, gap):
    """Only the small weights count.  Each is off by up to 2^-36 of the largest, by
    itself: 2^-36 / sqrt(3) sqrt(sum v^2) as a deviation, six of which no output
    passes, beside the module's relative bar."""
    tt.say("tree, one key far above, no value", dim, fmt, gap)
    b = Sink(device, oracle, dim, 32768, gap, fmt == "q8_0", sink_value=0.0)
    want = b.want()
    floor = 6 * 2.0 ** -36 / np.sqrt(3) * np.sqrt(np.square(b.v.astype(np.float64)).sum(0).max())
    for rows in ROWS:
        monkeypatch.setenv("TVARA_TREE_ROWS", rows)
        off = np.abs(b.run("f32x3") - want)
        assert (off <= floor + tt.BAR * np.abs(want).max()).all(), (off.max(), np.abs(want).max())


@pytest.mark.parametrize("bad", [65520.0, -1e5, 3e6, -3e38, np.nan, np.inf])
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
@pytest.mark.parametrize("dim", [64, 128])
def test_unseen_values_beyond_the_parts(device, oracle, monkeypatch, dim, fmt, bad):
    """f32x3: a node's value that fp16 does not hold leaves the rows that do not see it
    to the bit as they are, and is reported for those that do."""
    tt.say("tree, unseen beyond fp16", dim, fmt, bad)
    trees = [[-1, 0, 1, 1, 0, 4], tt.chain(2), [-1] * 20 + [3] * 20]
    for rows in ROWS:
        monkeypatch.setenv("TVARA_TREE_ROWS", rows)
        b = tt.Batch(device, oracle, 4, 2, dim, [35, 20, 700], trees, q8=fmt == "q8_0", seed=8)
        clean = b.run("f32x3")
        tt.agree(clean, b.want(), "f32x3")
        b.tv[4, 3] = b.tv[8 + 3, dim + 5] = bad  # seen by rows 4, 5 of the first tree; 3 and 20 to 39 of the third
        hit = np.array([4, 5, 8 + 3, *range(8 + 20, 8 + 40)])
        keep = np.setdiff1d(np.arange(b.rows), hit)
        with tt.hip_rows(b) as d:
            plan = attention.TreePlan(b.cache, b.seqs, b.nodes, b.parents, 4, 1 << 20, precision="f32x3")
            plan.launch(0, d.q.ptr, d.k.ptr, d.v.ptr, d.out.ptr)
            with pytest.raises(_capi.InvalidArgument, match="invalid online attention input"):
                plan.check()
            got = d.out.numpy()[: b.rows]
        assert np.array_equal(got[keep], clean[keep])
        heads = got[hit].reshape(hit.size, 4, dim)
        assert not np.isfinite(heads[:2, :2, 3]).any() and not np.isfinite(heads[2:, 2:, 5]).any()
        other = np.isfinite(got[hit]).sum()
        assert other == got[hit].size - 2 * hit.size  # one column of the two heads of that KV head


@pytest.mark.parametrize("dim", [64, 128])
def test_largest_values_of_the_parts(device, oracle, monkeypatch, dim):
    """f32x3 takes values up to fp16's own range."""
    tt.say("tree, largest values of fp16", dim)
    for rows in ROWS:
        monkeypatch.setenv("TVARA_TREE_ROWS", rows)
        b = tt.Batch(device, oracle, 4, 2, dim, [35, 700], [tt.bushy(6, 2), [-1] * 20], seed=9)
        b.tv[3, 7], b.tv[8, 2] = 65519.0, -65519.0
        tt.agree(b.run("f32x3"), b.want(), "f32x3")


@pytest.mark.parametrize("gap", [0.5, 12, 21])
@pytest.mark.parametrize("dim", [32, 96])
def test_long_sums_of_the_row_kernel(device, oracle, monkeypatch, dim, gap):
    """Layouts without tiles: as many waves as take a whole context each."""
    tt.say("tree, rows, long sums", dim, gap)
    monkeypatch.setattr(Sink, "TREES", 1024)
    b = Sink(device, oracle, dim, 32768, gap, False)
    tt.agree(b.run("f32"), b.want(), "f32")


@pytest.mark.parametrize("size", [1e4, 100.0, 0.01, 1e-3, 1e-4])
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
@pytest.mark.parametrize("dim", [64, 128])
def test_sizes_of_values(device, oracle, monkeypatch, dim, fmt, size):
    """f32 is as near at any size.  f32x3 holds a value to 2^-25 at the finest, off by
    2^-25 / sqrt(3) as a deviation: outputs are the same means of values and of their
    roundings, which are independent, so that they are off by 2^-25 / (sqrt(3) size)
    more, here with half as much again for outputs that happen to be small."""
    tt.say("tree, sizes of values", dim, fmt, size)
    b = tt.Batch(device, oracle, 8, 2, dim, [300, 33, 1500], [tt.bushy(12, 4), tt.chain(20), tt.bushy(40, 9)], seed=dim, layers=1)
    w, q8 = b.w, fmt == "q8_0"
    b.cache = device.PagedCache(1, 2, dim, 16, 200, fmt=device.Q8_0 if q8 else device.F32)
    b.seqs = []
    for i, n in enumerate(b.lengths):
        k, v = b.k[i], np.ascontiguousarray(b.v[i] * size, np.float32)
        b.seqs.append(b.cache.create_sequence())
        b.cache.append_many(b.seqs[i], k, v)
        if q8:
            k, v = (oracle.dequantize_q8_0(oracle.quantize_q8_0(np.ascontiguousarray(x, np.float32))).reshape(n, w) for x in (k, v))
        b.k[i], b.v[i] = k, v
    b.tv = np.ascontiguousarray(b.tv * size, np.float32)
    want = b.want()
    bars = {"f32": tt.NORM["f32"], "f32x3": tt.NORM["f32x3"] + 1.5 * 2.0 ** -25 / (np.sqrt(3) * size)}
    for precision, rows in [("f32", "")] + [("f32x3", r) for r in ROWS]:
        monkeypatch.setenv("TVARA_TREE_ROWS", rows)
        off = np.linalg.norm(b.run(precision) - want) / np.linalg.norm(want)
        assert off <= bars[precision], (precision, rows, off)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("dim", [64, 128])
def test_sizes_of_keys(device, oracle, monkeypatch, dim, rows):
    """Keys of 70 beside queries of 1/70: the scores are those of N(0,1), each off by
    2^-25 / sqrt(3) * 70 sqrt(dim) * ln 2 as a deviation, 1e-5, which the mean of a
    row's values is off by less than."""
    tt.say("tree, sizes of keys", dim, rows)
    monkeypatch.setenv("TVARA_TREE_ROWS", rows)
    b = tt.Batch(device, oracle, 8, 2, dim, [300, 33], [tt.bushy(12, 4), tt.chain(20)], seed=dim, scale=70.0)
    b.q = np.ascontiguousarray(b.q / 70, np.float32)
    tt.agree(b.run("f32x3"), b.want(), "f32x3")
