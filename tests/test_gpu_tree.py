"""Trees of drafted tokens over the paged cache on the GPU: their attention,
greedy acceptance, slot maps with block tables, the write of accepted rows, and
one step of them together, against plain implementations in 64 bits.

Attention bars.  f32: a score is d products and sums of f32 operands, off by at
most (d + 2) 2^-24 sum_i |q_i k_i| / sqrt(d); for N(0,1) inputs at d <= 256
sum_i |q_i k_i| / sqrt(d) <= 0.8 sqrt(d) < 13, so a probability is off by less
than 258 * 2^-24 * 13 = 2e-4 relative in that worst case and sqrt(258) 2^-24 13 =
1.3e-5 as independent roundings go; an output is a mean of such terms around its
own value, |v - o| <= 10, n_eff of them: 1e-4 * (1 + |ref|) holds the typical
error eightfold.  In the 2-norm, over many outputs, the roundings are
independent: 2e-6 relative.  f32x3: scores carry 2^-22 per product (fp16 parts);
for values and probabilities in two parts of 8 bits each, the second rounded to
nearest, 2^-17 * sqrt(2) / sqrt(3) = 6.2e-6 of a term's size as independent
roundings; terms may cancel down to 1/2 of the output: the same 1e-4 and 1.3e-5
(in fp16 parts, as they are, they are off by less).
Whole numbers and stored bytes are equal.
"""

import ctypes as C
import sys

import numpy as np
import pytest

import refmath
from tvara_amd import _capi, attention, hip, synth
from tvara_amd.kv import SlotPlan

pytestmark = pytest.mark.gpu
BAR = 1e-4
NORM = {"f32": 2e-6, "f32x3": 1.3e-5}


def say(*a):
    print(*a, flush=True, file=sys.stderr)


def chain(n):
    return list(range(-1, n - 1))


def bushy(n, width, seed=0, roots=0.1):
    r = np.random.default_rng(seed)
    return [-1 if j == 0 or r.random() < roots else int(r.integers(max(0, j - width), j)) for j in range(n)]


def ancestors(parents):
    seen = np.zeros((len(parents), len(parents)), bool)
    for j, p in enumerate(parents):
        if p >= 0:
            seen[j] = seen[p]
        seen[j, j] = True
    return seen


class Batch:
    """Sequences of the given lengths with a tree each, on the GPU and in plain arrays."""

    def __init__(self, device, oracle, heads, kv_heads, dim, lengths, trees, tpb=16, q8=False, seed=1, layers=1, spare=0,
                 scale=1.0):
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.lengths, self.trees, self.layers = list(lengths), [list(t) for t in trees], layers
        w = self.w = kv_heads * dim
        blocks = sum(-(-n // tpb) for n in lengths) + spare + 1
        self.cache = device.PagedCache(layers, kv_heads, dim, tpb, blocks, fmt=device.Q8_0 if q8 else device.F32)
        self.seqs, self.k, self.v = [], [], []
        for i, n in enumerate(lengths):
            k = scale * synth.normal(seed, f"k{i}", max(1, n * layers * w))[: n * layers * w].reshape(n, layers * w)
            v = synth.normal(seed, f"v{i}", max(1, n * layers * w))[: n * layers * w].reshape(n, layers * w)
            s = self.cache.create_sequence()
            if n:
                self.cache.append_many(s, k, v)
            if q8 and n:
                k, v = (oracle.dequantize_q8_0(oracle.quantize_q8_0(x)).reshape(n, layers * w) for x in (k, v))
            self.seqs.append(s)
            self.k.append(k)
            self.v.append(v)
        self.nodes = [len(t) for t in trees]
        self.parents = [p for t in trees for p in t]
        rows = self.rows = len(self.parents)
        self.q = synth.normal(seed, "q", max(1, rows * heads * dim))[: rows * heads * dim].reshape(rows, heads * dim)
        self.tk = scale * synth.normal(seed, "tk", max(1, rows * w))[: rows * w].reshape(rows, w)
        self.tv = synth.normal(seed, "tv", max(1, rows * w))[: rows * w].reshape(rows, w)

    def run(self, precision="f32", visible=None, layer=0):
        return attention.tree_batch(self.cache, self.q, self.seqs, self.nodes, self.parents, self.tk, self.tv, layer,
                                    self.heads, 1 << 20, visible=visible, precision=precision)

    def want(self, visible=None, layer=0):
        out, r0 = np.empty((self.rows, self.heads * self.dim)), 0
        cols = slice(layer * self.w, (layer + 1) * self.w)
        for i, t in enumerate(self.trees):
            n = self.lengths[i] if visible is None else min(self.lengths[i], int(np.broadcast_to(visible, len(self.trees))[i]))
            seen = ancestors(t)
            for j in range(len(t)):
                on = np.flatnonzero(seen[j]) + r0
                out[r0 + j] = refmath.attention(self.q[r0 + j], np.concatenate([self.k[i][:n, cols], self.tk[on]]),
                                                np.concatenate([self.v[i][:n, cols], self.tv[on]]), self.heads,
                                                self.kv_heads, self.dim)
            r0 += len(t)
        return out


def agree(got, want, precision):
    got = np.asarray(got, np.float64)
    assert np.isfinite(got).all()
    assert refmath.close(got, want, BAR), refmath.max_rel(got, want)
    if want.size:
        off = np.linalg.norm(got - want) / np.linalg.norm(want)
        assert off <= NORM[precision], off


PRECISIONS = ["f32", "f32x3"]


@pytest.mark.parametrize("precision", PRECISIONS)
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 7, 8, 10, 16])
def test_groups(device, oracle, group, dim, fmt, precision):
    say("tree groups", group, dim, fmt, precision)
    trees = [chain(3), bushy(9, 3), bushy(17, 6), [-1]]
    b = Batch(device, oracle, 2 * group, 2, dim, [137, 64, 20, 1], trees, q8=fmt == "q8_0", seed=group)
    agree(b.run(precision), b.want(), precision)


@pytest.mark.parametrize("precision", PRECISIONS)
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 500])
def test_lengths(device, oracle, length, fmt, precision):
    say("tree lengths", length, fmt, precision)
    trees = [bushy(5, 2), chain(1), [], bushy(33, 9), [-1] * 4]
    b = Batch(device, oracle, 8, 2, 64, [length, length + 3, 7, length, 0], trees, q8=fmt == "q8_0", seed=length)
    agree(b.run(precision), b.want(), precision)


@pytest.mark.parametrize("precision", PRECISIONS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("nodes", [1, 2, 4, 16, 31, 32, 33, 64, 65, 100, 257])
def test_tree_sizes(device, oracle, nodes, dim, precision):
    say("tree sizes", nodes, dim, precision)
    trees = [bushy(nodes, 7, seed=nodes), chain(nodes), [-1] * min(nodes, 40)]
    b = Batch(device, oracle, 4, 1, dim, [90, 33, 200], trees, seed=nodes)
    agree(b.run(precision), b.want(), precision)


@pytest.mark.parametrize("precision", PRECISIONS)
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
@pytest.mark.parametrize("dim,tpb", [(64, 32), (64, 64), (128, 128), (128, 1024), (64, 2048), (64, 8), (64, 48), (128, 1),
                                     (32, 16), (96, 16), (256, 16), (512, 16)])
def test_layouts(device, oracle, dim, tpb, fmt, precision):
    """Blocks and head_dims with tiles and without."""
    say("tree layouts", dim, tpb, fmt, precision)
    b = Batch(device, oracle, 6, 2, dim, [333, 100, 47], [bushy(11, 4), bushy(6, 2), chain(2)], tpb=tpb,
              q8=fmt == "q8_0", seed=dim + tpb)
    agree(b.run(precision), b.want(), precision)


@pytest.mark.parametrize("precision", PRECISIONS)
@pytest.mark.parametrize("heads,kv_heads,dim,tpb", [(2, 1, 2, 16), (3, 3, 10, 4), (4, 2, 66, 16), (5, 5, 64, 16)])
def test_odd_shapes(device, oracle, heads, kv_heads, dim, tpb, precision):
    say("tree odd shapes", heads, kv_heads, dim, tpb, precision)
    b = Batch(device, oracle, heads, kv_heads, dim, [50, 9], [bushy(5, 4), chain(3)], tpb=tpb, seed=dim)
    agree(b.run(precision), b.want(), precision)


@pytest.mark.parametrize("precision", PRECISIONS)
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
@pytest.mark.parametrize("dim", [64, 128])
def test_long_contexts(device, oracle, dim, fmt, precision):
    """Keys in many runs; a few rows of the batch are checked."""
    say("tree long contexts", dim, fmt, precision)
    b = Batch(device, oracle, 8, 2, dim, [9001, 130, 20000], [bushy(12, 4), chain(4), bushy(3, 2)], tpb=64,
              q8=fmt == "q8_0", seed=3)
    got, want = b.run(precision), b.want()
    agree(got, want, precision)


@pytest.mark.parametrize("precision", PRECISIONS)
def test_sharp_scores(device, oracle, precision):
    """Scores that spread over tens of units, the maximum anywhere."""
    say("tree sharp scores", precision)
    b = Batch(device, oracle, 8, 2, 128, [700, 65], [bushy(20, 5), bushy(9, 3)], seed=12, scale=4.0)
    got, want = b.run(precision), b.want()
    # scores of sigma 4: four times the score error of the module's bar
    assert refmath.close(got, want, 4 * BAR), refmath.max_rel(got, want)


@pytest.mark.parametrize("precision", PRECISIONS)
@pytest.mark.parametrize("dim", [64, 96])
def test_visible(device, oracle, dim, precision):
    say("tree visible", dim, precision)
    b = Batch(device, oracle, 4, 2, dim, [100, 64, 40], [bushy(7, 3), chain(2), bushy(3, 3)], seed=5)
    visible = np.array([37, 0, 1000])
    agree(b.run(precision, visible), b.want(visible), precision)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("precision", PRECISIONS)
@pytest.mark.parametrize("dim", [64, 128, 96])
def test_what_is_not_seen_does_not_count(device, oracle, dim, precision, bad):
    """Nodes whose keys or values are not finite reach only the rows that see
    them; stale slots behind a sequence's end reach none."""
    say("tree unseen", dim, precision, bad)
    tree = [-1, 0, 1, 1, 0, 4]  # node 4's K/V are bad: nodes 4 and 5 see them
    b = Batch(device, oracle, 4, 2, dim, [35, 20], [tree, chain(2)], seed=8)
    s = b.seqs[0]
    big = np.full((1, b.w), 3e38, np.float32)
    for _ in range(3):
        b.cache.append(s, big * 10, big * np.nan)
    b.cache.truncate(s, 35)
    want = b.want()
    clean = b.run(precision)
    agree(clean, want, precision)
    b.tv[4] = bad
    keep = [0, 1, 2, 3, 6, 7]
    if precision == "f32":
        got = b.run(precision)
        assert np.array_equal(got[keep], clean[keep])
        assert not np.isfinite(got[4:6]).any()
    else:
        _untouched(b, precision, clean, keep, None)
    b.tk[4] = bad
    _untouched(b, precision, clean, keep, "invalid online attention input")


def _untouched(b, precision, clean, keep, message):
    """A launch that may fail its check: the rows of `keep` are as without the bad node."""
    with hip_rows(b) as d:
        plan = attention.TreePlan(b.cache, b.seqs, b.nodes, b.parents, b.heads, 1 << 20, precision=precision)
        plan.launch(0, d.q.ptr, d.k.ptr, d.v.ptr, d.out.ptr)
        try:
            plan.check()
            assert message is None
        except _capi.InvalidArgument as e:
            assert message is None or message in str(e)
        assert np.array_equal(d.out.numpy()[keep], clean[keep])


class hip_rows:
    def __init__(self, b, stride=None):
        self.q = hip.DeviceArray.from_numpy(b.q.astype(np.float32))
        k, v = b.tk.astype(np.float32), b.tv.astype(np.float32)
        if stride:
            k, v = (np.concatenate([x, np.full((b.rows, stride - b.w), np.nan, np.float32)], 1) for x in (k, v))
        self.k, self.v = hip.DeviceArray.from_numpy(k), hip.DeviceArray.from_numpy(v)
        self.out = hip.DeviceArray.from_numpy(np.full((b.rows + 2, b.heads * b.dim), 7.0, np.float32))

    def __enter__(self):
        return self

    def __exit__(self, *a):
        hip.synchronize()


@pytest.mark.parametrize("precision", PRECISIONS)
@pytest.mark.parametrize("dim,tpb", [(64, 16), (128, 16), (96, 16), (64, 8)])
def test_plan_strides_and_layers(device, oracle, dim, tpb, precision):
    """Node rows with a stride, every layer, rows behind the last left as they
    were; a plan fails once the cache has changed."""
    say("tree plan", dim, tpb, precision)
    b = Batch(device, oracle, 6, 2, dim, [77, 16, 0], [bushy(10, 3), [], chain(4)], tpb=tpb, layers=3, seed=21)
    with hip_rows(b, stride=b.w + 12) as d:
        plan = attention.TreePlan(b.cache, b.seqs, b.nodes, b.parents, b.heads, 1 << 20, precision=precision)
        for layer in range(3):
            plan.launch(layer, d.q.ptr, d.k.ptr, d.v.ptr, d.out.ptr, row_stride=b.w + 12)
            plan.check()
            got = d.out.numpy()
            agree(got[: b.rows], b.want(layer=layer), precision)
            assert (got[b.rows:] == 7).all()
            assert np.array_equal(got[: b.rows], b.run(precision, layer=layer))
        for bad in (lambda: plan.launch(3, d.q.ptr, d.k.ptr, d.v.ptr, d.out.ptr),
                    lambda: plan.launch(0, d.q.ptr, d.k.ptr, d.v.ptr, d.out.ptr, row_stride=b.w - 4),
                    lambda: plan.launch(0, d.q.ptr, d.k.ptr, d.v.ptr, d.out.ptr, row_stride=b.w + 1),
                    lambda: plan.launch(0, d.q.ptr, d.k.ptr, d.v.ptr, d.out.ptr, row_stride=(1 << 23) + 4),
                    lambda: plan.launch(0, d.q.ptr, d.k.ptr, d.v.ptr, d.out.ptr, row_stride=1 << 62),
                    lambda: plan.launch(0, d.q.ptr + 4, d.k.ptr, d.v.ptr, d.out.ptr)):
            with pytest.raises(_capi.InvalidArgument):
                bad()
        b.cache.truncate(b.seqs[0], 70)
        with pytest.raises(_capi.InvalidArgument, match="stale"):
            plan.launch(0, d.q.ptr, d.k.ptr, d.v.ptr, d.out.ptr)


@pytest.mark.parametrize("nodes", [3, 12, 40])
@pytest.mark.parametrize("where", ["q", "cached keys", "cached values", "keys", "values"])
@pytest.mark.parametrize("q8", [False, True])
def test_beyond_fp16_is_reported(device, oracle, where, nodes, q8):
    """f32x3 reports inputs that its fp16 parts do not hold; f32 takes them."""
    say("tree beyond fp16", where, nodes, q8)
    b = Batch(device, oracle, 8, 2, 64, [70], [chain(nodes)], seed=3, spare=1)
    if where.startswith("cached"):
        if q8:  # (a Q8_0 element is at most 127 * 65,504: the scales are fp16)
            b = Batch(device, oracle, 8, 2, 64, [70], [chain(nodes)], seed=3, spare=1, q8=True)
        row = [np.array(x[0][69:70], np.float64) for x in (b.k, b.v)]
        row["keys" not in where][:, 5] = 3e5
        b.cache.truncate(b.seqs[0], 69)
        b.cache.append(b.seqs[0], *(np.ascontiguousarray(x) for x in row))
    else:
        x = b.q if where == "q" else b.tk if where == "keys" else b.tv
        x[0, 5] = 3e6
    message = None
    try:
        b.run("f32x3")
    except _capi.InvalidArgument as e:
        message = str(e)
    assert message == "invalid online attention input"
    assert np.isfinite(b.run("f32")).all()


@pytest.mark.parametrize("precision", PRECISIONS)
def test_launches_repeat_to_the_bit(device, oracle, precision):
    """Runs of a long context and their merge, one launch after the other in one plan."""
    say("tree launches repeat", precision)
    b = Batch(device, oracle, 8, 2, 64, [3000, 100], [bushy(9, 3), chain(30)], seed=6)
    with hip_rows(b) as d:
        plan = attention.TreePlan(b.cache, b.seqs, b.nodes, b.parents, b.heads, 1 << 20, precision=precision)
        first = None
        for _ in range(6):
            d.out.zero()
            plan.launch(0, d.q.ptr, d.k.ptr, d.v.ptr, d.out.ptr)
            plan.check()
            got = d.out.numpy()
            first = got if first is None else first
            assert np.array_equal(got, first)
        agree(first[: b.rows], b.want(), precision)


def test_one_sequence_in_several_trees(device, oracle):
    say("tree of one sequence twice")
    b = Batch(device, oracle, 8, 2, 64, [150], [bushy(8, 3)], seed=4)
    twice = attention.tree_batch(b.cache, np.concatenate([b.q, b.q]), b.seqs * 2, b.nodes * 2, b.parents * 2,
                                 np.concatenate([b.tk, b.tk]), np.concatenate([b.tv, b.tv]), 0, 8, 1 << 20)
    one = b.want()
    agree(twice, np.concatenate([one, one]), "f32")


def test_chain_is_the_prompt_chunk(device, oracle):
    """A chain of nodes attends as the same tokens of a prompt chunk do."""
    say("tree chain against prompt chunk")
    b = Batch(device, oracle, 8, 2, 64, [100], [chain(12)], seed=14, spare=2)
    got = b.run()
    b.cache.append_many(b.seqs[0], b.tk, b.tv)
    chunk = attention.prefill_batch(b.cache, b.q, b.seqs, [100], [12], 0, 8, 1 << 20)
    assert refmath.close(got, chunk, BAR)


@pytest.mark.parametrize("rows", ["16", "32", "128"])
class TestRowBlocks:
    """Each number of rows that a workgroup of f32x3 may have, whatever the batch."""

    @pytest.fixture(autouse=True)
    def choose(self, monkeypatch, rows):
        monkeypatch.setenv("TVARA_TREE_ROWS", rows)

    @pytest.mark.parametrize("fmt", ["f32", "q8_0"])
    @pytest.mark.parametrize("dim", [64, 128])
    @pytest.mark.parametrize("group", [1, 3, 4, 8])
    def test_groups(self, device, oracle, rows, group, dim, fmt):
        test_groups(device, oracle, group, dim, fmt, "f32x3")

    @pytest.mark.parametrize("fmt", ["f32", "q8_0"])
    @pytest.mark.parametrize("length", [0, 1, 16, 31, 32, 33, 300])
    def test_lengths(self, device, oracle, rows, length, fmt):
        test_lengths(device, oracle, length, fmt, "f32x3")

    @pytest.mark.parametrize("dim", [64, 128])
    @pytest.mark.parametrize("nodes", [1, 8, 31, 33, 65, 200])
    def test_tree_sizes(self, device, oracle, rows, nodes, dim):
        test_tree_sizes(device, oracle, nodes, dim, "f32x3")

    @pytest.mark.parametrize("fmt", ["f32", "q8_0"])
    @pytest.mark.parametrize("dim,tpb", [(64, 32), (128, 16), (128, 128), (64, 2048)])
    def test_layouts(self, device, oracle, rows, dim, tpb, fmt):
        test_layouts(device, oracle, dim, tpb, fmt, "f32x3")

    @pytest.mark.parametrize("dim", [64, 128])
    def test_long_contexts_strides_and_visible(self, device, oracle, rows, dim):
        test_long_contexts(device, oracle, dim, "f32", "f32x3")
        test_long_contexts(device, oracle, dim, "q8_0", "f32x3")
        test_plan_strides_and_layers(device, oracle, dim, 16, "f32x3")
        test_visible(device, oracle, dim, "f32x3")
        test_sharp_scores(device, oracle, "f32x3")

    @pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
    @pytest.mark.parametrize("dim", [64, 128])
    def test_what_is_not_seen_does_not_count(self, device, oracle, rows, dim, bad):
        test_what_is_not_seen_does_not_count(device, oracle, dim, "f32x3", bad)

    @pytest.mark.parametrize("where", ["q", "cached keys", "cached values", "keys", "values"])
    @pytest.mark.parametrize("q8", [False, True])
    def test_beyond_fp16_is_reported(self, device, oracle, rows, where, q8):
        test_beyond_fp16_is_reported(device, oracle, where, 12, q8)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("trees", [12, 70, 300])
def test_rows_by_the_batch(device, oracle, trees, dim):
    """Batches of few, of more and of many short trees, which take other rows a workgroup."""
    say("tree rows by the batch", trees, dim)
    lengths = [(7 * i) % 50 for i in range(trees)]
    b = Batch(device, oracle, 8, 2, dim, lengths, [bushy(1 + i % 17, 4, seed=i) for i in range(trees)], seed=trees)
    agree(b.run("f32x3"), b.want(), "f32x3")
    agree(b.run("f32"), b.want(), "f32")


@pytest.mark.parametrize("precision,rows", [("f32", ""), ("f32x3", "16"), ("f32x3", "32"), ("f32x3", "128")])
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
@pytest.mark.parametrize("dim", [64, 128])
def test_long_runs(device, oracle, monkeypatch, dim, fmt, precision, rows):
    """Enough trees that a workgroup walks a long context alone, through a table of
    blocks in no order: one sequence of 16,003 tokens under 500 trees of a node."""
    say("tree long runs", dim, fmt, precision, rows)
    monkeypatch.setenv("TVARA_TREE_ROWS", rows)
    n, trees, heads, w = 16003, 500, 4, 2 * dim
    cache = device.PagedCache(1, 2, dim, 16, 1800, fmt=device.Q8_0 if fmt == "q8_0" else device.F32)
    k, v = (synth.normal(dim, x, n * w).reshape(n, w) for x in "kv")
    a, b = cache.create_sequence(), cache.create_sequence()
    for i in range(0, n, 48):  # the other sequence's blocks lie between
        cache.append_many(a, k[i:i + 48], v[i:i + 48])
        cache.append_many(b, k[:16 * (1 + i // 48 % 2)], v[:16 * (1 + i // 48 % 2)])
    if fmt == "q8_0":
        k, v = (oracle.dequantize_q8_0(oracle.quantize_q8_0(x)).reshape(n, w) for x in (k, v))
    q, tk, tv = (synth.normal(dim, x, trees * c).reshape(trees, c) for x, c in (("q", heads * dim), ("tk", w), ("tv", w)))
    got = attention.tree_batch(cache, q, [a] * trees, [1] * trees, [-1] * trees, tk, tv, 0, heads, 1 << 20, precision=precision)
    want = np.empty((trees, heads, dim))
    for h in range(heads):
        cols = slice(h // 2 * dim, (h // 2 + 1) * dim)
        x = q.reshape(trees, heads, dim)[:, h].astype(np.float64)
        s = np.concatenate([x @ k[:, cols].astype(np.float64).T, (x * tk[:, cols]).sum(1, keepdims=True)], 1) / np.sqrt(dim)
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        want[:, h] = p[:, :n] @ v[:, cols].astype(np.float64) + p[:, n:] * tv[:, cols]
    agree(got, want.reshape(trees, heads * dim), precision)


@pytest.mark.parametrize("dim,kv_heads", [(128, 8), (64, 16), (96, 10)])
def test_pool_beyond_32_bits(device, oracle, monkeypatch, dim, kv_heads):
    """Blocks more than 4 GiB into the pool: attention, slots, writes."""
    say("tree, pool beyond 4 GiB", dim)
    w, heads, n = kv_heads * dim, 2 * kv_heads, 100
    per = (5 << 30) // (16 * w * 8) + 1
    cache = device.PagedCache(1, kv_heads, dim, 16, per + 20)
    filler, a = cache.create_sequence(), cache.create_sequence()
    cache.reserve([filler], [16 * per])
    k, v = (synth.normal(dim, x, n * w).reshape(n, w) for x in "kv")
    cache.reserve([a], [n])
    up = hip.DeviceArray.from_numpy
    base, stride = cache.pool_address()
    assert min(h[0] for h in cache.blocks(a)) * stride > 1 << 32
    plan = SlotPlan(cache, [a])
    slots, starts, counts = hip.DeviceArray((n,), np.int64), up(np.zeros(1, np.int32)), up(np.full(1, n, np.int32))
    plan.build(starts.ptr, counts.ptr, 0, n, slots_ptr=slots.ptr)
    dk, dv = up(k.astype(np.float32)), up(v.astype(np.float32))
    plan.write(slots.ptr, None, n, dk.ptr, dv.ptr, n, w, w)
    plan.check()
    assert np.array_equal(cache.read_all(a, 0).reshape(n, w), k.astype(np.float32))
    q, tk, tv = (synth.normal(dim, x, 2 * c).reshape(2, c) for x, c in (("q", heads * dim), ("tk", w), ("tv", w)))
    want = np.empty((2, heads, dim))
    for h in range(heads):
        cols = slice(h // 2 * dim, (h // 2 + 1) * dim)
        for r in range(2):  # node 1 sees node 0 and itself
            kk = np.concatenate([k[:, cols], tk[: r + 1, cols]]).astype(np.float64)
            vv = np.concatenate([v[:, cols], tv[: r + 1, cols]]).astype(np.float64)
            s = kk @ q[r].reshape(heads, dim)[h].astype(np.float64) / np.sqrt(dim)
            p = np.exp(s - s.max())
            want[r, h] = p @ vv / p.sum()
    for precision, rows in (("f32", ""), ("f32x3", "16"), ("f32x3", "32"), ("f32x3", "128")):
        monkeypatch.setenv("TVARA_TREE_ROWS", rows)
        got = attention.tree_batch(cache, q, [a], [2], [-1, 0], tk, tv, 0, heads, 1 << 20, precision=precision)
        agree(got, want.reshape(2, heads * dim), precision)


@pytest.mark.parametrize("bad", [None, np.nan, np.inf])
@pytest.mark.parametrize("fmt,most", [("f32", 340), ("q8_0", 90)])
@pytest.mark.parametrize("dim", [64, 128])
def test_many_short_trees(device, oracle, dim, fmt, most, bad):
    """Batches whose waves work on their own; values that few nodes see."""
    say("many short trees", dim, fmt, bad)
    trees = [[-1, 0, 0, 1] if i % 50 == 7 else bushy(1 + i % 21, 4, seed=i) for i in range(360)]
    b = Batch(device, oracle, 8, 2, dim, [(37 * i) % most for i in range(360)], trees, q8=fmt == "q8_0", seed=dim)
    want, clean = b.want(), b.run("f32")
    agree(clean, want, "f32")
    if bad is None:
        with hip_rows(b) as d:  # (rows behind the last stay)
            plan = attention.TreePlan(b.cache, b.seqs, b.nodes, b.parents, b.heads, 1 << 20)
            plan.launch(0, d.q.ptr, d.k.ptr, d.v.ptr, d.out.ptr)
            plan.check()
            assert np.array_equal(d.out.numpy()[: b.rows], clean) and (d.out.numpy()[b.rows:] == 7).all()
        return
    hit = [sum(map(len, trees[:i])) + 2 for i in range(7, 360, 50)]  # node 2 of such a tree: only it sees itself
    b.tv[hit] = bad
    got = b.run("f32")
    keep = np.setdiff1d(np.arange(b.rows), hit)
    assert np.array_equal(got[keep], clean[keep]) and not np.isfinite(got[hit]).any()


def test_tree_refusals(device, oracle):
    say("tree refusals")
    b = Batch(device, oracle, 4, 2, 64, [20, 5], [chain(3), [-1, 0]], seed=2)

    def plan(**kw):
        a = dict(seqs=b.seqs, nodes=b.nodes, parents=b.parents, heads=4, context=1 << 20)
        a.update(kw)
        return attention.TreePlan(b.cache, **a)

    for kw in (dict(parents=[-1, 0, 2, -1, 0]), dict(parents=[-1, 0, 1, 0, 0]), dict(parents=[-2, 0, 1, -1, 0]),
               dict(nodes=[2, 2]), dict(seqs=[b.seqs[0], 99]), dict(heads=3), dict(heads=0), dict(context=22),
               dict(context=10), dict(precision="bf16"), dict(precision="f16"), dict(seqs=[], nodes=[], parents=[]),
               dict(nodes=[1025, 0], parents=chain(1025))):
        with pytest.raises(_capi.InvalidArgument):
            plan(**kw)
    plan(context=23).close()
    plan(nodes=[0, 0], parents=[]).close()
    assert attention.tree_batch(b.cache, np.zeros((0, 256)), b.seqs, [0, 0], [], np.zeros((0, 128)),
                                np.zeros((0, 128)), 0, 4, 1 << 20).shape == (0, 256)


# ------------------------------------------------------------- acceptance

def walk(parents, tokens, first, logits):
    """The definition, a step at a time: (path, next)."""
    at, want, path = -1, int(first), []
    while True:
        child = next((j for j, p in enumerate(parents) if p == at and tokens[j] == want), None)
        if child is None:
            return path, want
        path.append(child)
        at = child
        row = np.where(np.isnan(logits[child]), -np.inf, logits[child])
        order = np.isnan(logits[child]).all()
        want = 0 if order else int(np.argmax(row))


def accept(device, trees, tokens, first, logits, path_stride, logits_stride=0, stream=None, check=True):
    cache = device.PagedCache(1, 1, 64, 16, 1)
    seqs = [cache.create_sequence() for _ in trees]
    plan = attention.TreePlan(cache, seqs, [len(t) for t in trees], [p for t in trees for p in t], 1, 4096)
    up = hip.DeviceArray.from_numpy
    n = len(trees)
    dt, df = up(np.asarray(tokens + [0], np.uint32)), up(np.asarray(first, np.uint32))
    rows = np.asarray(logits, np.float32)
    vocab = rows.shape[1]
    if logits_stride:
        rows = np.concatenate([rows, np.full((rows.shape[0], logits_stride - vocab), 1e30, np.float32)], 1)
    dl = up(rows)
    path = up(np.full((n + 1, max(1, path_stride)), 77, np.int32))
    acc, nxt = up(np.full(n + 1, 77, np.int32)), up(np.full(n + 1, 77, np.uint32))
    plan.accept(dt.ptr, df.ptr, dl.ptr, vocab, path.ptr, path_stride, acc.ptr, nxt.ptr, logits_stride=logits_stride)
    hip.synchronize()
    assert (path.numpy()[n] == 77).all() and acc.numpy()[n] == 77 and nxt.numpy()[n] == 77
    if check:
        plan.check()
    return plan, path.numpy()[:n], acc.numpy()[:n], nxt.numpy()[:n]


@pytest.mark.parametrize("vocab,stride", [(1, 0), (2, 0), (37, 40), (1000, 0), (2049, 0), (32000, 32004), (128256, 0)])
@pytest.mark.parametrize("sizes", [[1], [5, 0, 33, 100], [8] * 40])
def test_acceptance(device, vocab, stride, sizes):
    if vocab == 128256 and sum(sizes) > 200:
        sizes = sizes[:10]
    say("acceptance", vocab, stride, sizes)
    r = np.random.default_rng(vocab + len(sizes))
    trees = [bushy(n, 3, seed=i, roots=0.2) for i, n in enumerate(sizes)]
    total = sum(sizes)
    logits = np.round(r.normal(size=(max(total, 1), vocab)) * 2).astype(np.float32)  # many ties
    tokens, first, at = [], [], 0
    for t in trees:
        mine = []
        for j, p in enumerate(t):
            agrees = r.random() < 0.8
            mine.append(int(np.argmax(logits[at + p])) if p >= 0 and agrees else int(r.integers(vocab)))
        first.append(mine[int(r.integers(len(mine)))] if mine and r.random() < 0.8 else int(r.integers(vocab)))
        tokens += mine
        at += len(t)
    _, path, acc, nxt = accept(device, trees, tokens, first, logits, 12, stride)
    at = 0
    for i, t in enumerate(trees):
        want, after = walk(t, tokens[at:at + len(t)], first[i], logits[at:at + len(t)])
        if len(want) <= 12:
            assert acc[i] == len(want) and nxt[i] == after
            assert path[i].tolist() == [at + j for j in want] + [-1] * (12 - len(want))
        at += len(t)


def test_acceptance_values(device):
    """Ties, signed zeros, infinities, rows of the lowest value, NaN."""
    say("acceptance values")
    low = np.finfo(np.float32).min
    rows = np.array([[0.0, -0.0, -1, -2], [-0.0, 0.0, -1, 0.0], [-np.inf, -np.inf, -np.inf, -np.inf], [low, low, -np.inf, low],
                     [1, np.inf, np.inf, 2], [-np.inf, low, -np.inf, -np.inf]], np.float32)
    best = [0, 0, 0, 0, 1, 1]
    trees = [[-1]] * len(rows)
    _, path, acc, nxt = accept(device, trees, [3] * len(rows), [3] * len(rows), rows, 2)
    assert acc.tolist() == [1] * len(rows) and nxt.tolist() == best
    plan, path, acc, nxt = accept(device, [[-1], [-1]], [3, 3], [3, 3],
                                  np.array([[1, np.nan, 2, 0], [np.nan, -np.inf, -1, np.nan]], np.float32), 2, check=False)
    assert nxt.tolist() == [2, 2] and acc.tolist() == [1, 1]
    with pytest.raises(_capi.InvalidArgument, match="logits"):
        plan.check()
    plan.check()  # reported once


def test_acceptance_path_without_room(device):
    say("acceptance without room")
    rows = np.eye(4, dtype=np.float32)
    plan, path, acc, nxt = accept(device, [chain(4)], [3, 0, 1, 2], [3], rows, 2, check=False)
    assert path.tolist() == [[0, 1]] and acc.tolist() == [2] and nxt.tolist() == [1]
    with pytest.raises(_capi.InvalidArgument, match="path"):
        plan.check()
    plan, path, acc, nxt = accept(device, [chain(4)], [3, 0, 1, 2], [9], rows, 0)
    assert acc.tolist() == [0] and nxt.tolist() == [9]


# ------------------------------------------------------------------ slots

def plain_map(cache, seqs, starts, counts, stride, capacity):
    b = cache.tokens_per_block
    refs = [[(h[0], cache.references(h)) for h in cache.blocks(s)] for s in seqs]
    offsets = np.concatenate([[0], np.cumsum(np.maximum(counts, 0))])
    pos, slots = np.full(capacity, -1), np.full(capacity, -1, np.int64)
    bad = False
    for i, (s, c) in enumerate(zip(starts, counts)):
        bad |= c < 0
        for j in range(max(c, 0)):
            at = i * stride + j if stride else offsets[i] + j
            if at >= capacity or (stride and j >= stride):
                bad = True
                continue
            pos[at] = s + j
            blk = (s + j) // b
            ok = s + j >= 0 and blk < len(refs[i]) and refs[i][blk][1] == 1
            bad |= not ok
            slots[at] = refs[i][blk][0] * b + (s + j) % b if ok else -1
    return offsets, pos, slots, bad


def built(cache, seqs, starts, counts, stride, capacity, width):
    up = hip.DeviceArray.from_numpy
    n = len(seqs)
    plan = SlotPlan(cache, seqs)
    ds, dc = up(np.asarray(starts, np.int32)), up(np.asarray(counts, np.int32))
    off, pos = up(np.full(n + 2, 77, np.int32)), up(np.full(capacity + 1, 77, np.int32))
    slots, tab = up(np.full(capacity + 1, 77, np.int64)), up(np.full((n + 1, max(1, width)), 77, np.int32))
    plan.build(ds.ptr, dc.ptr, stride, capacity, off.ptr, pos.ptr, slots.ptr, tab.ptr, width)
    hip.synchronize()
    assert off.numpy()[-1] == 77 and pos.numpy()[-1] == 77 and slots.numpy()[-1] == 77
    if width:
        assert (tab.numpy()[n:] == 77).all()
    return plan, off.numpy()[:-1], pos.numpy()[:-1], slots.numpy()[:-1], tab.numpy()[:n]


@pytest.mark.parametrize("tpb", [1, 4, 16, 48])
@pytest.mark.parametrize("n", [1, 3, 70, 300])
@pytest.mark.parametrize("stride", [0, 9])
def test_slot_map(device, n, tpb, stride):
    say("slot map", n, tpb, stride)
    r = np.random.default_rng(n * tpb)
    cache = device.PagedCache(1, 1, 2, tpb, n * (60 // tpb + 3))
    seqs = [cache.create_sequence() for _ in range(n)]
    lengths = r.integers(0, 50, n)
    for i in r.permutation(n):
        cache.reserve([seqs[i]], [lengths[i]])
    counts = r.integers(0, 10, n) if n > 1 else np.array([5])
    cache.reserve(seqs, counts)
    if stride:
        counts = np.minimum(counts, stride)
    capacity = n * stride + 3 if stride else int(counts.sum()) + 5
    width = max(len(cache.blocks(s)) for s in seqs) + 2
    plan, off, pos, slots, tab = built(cache, seqs, lengths, counts, stride, capacity, width)
    plan.check()
    woff, wpos, wslots, bad = plain_map(cache, seqs, lengths, counts, stride, capacity)
    assert not bad
    assert np.array_equal(off, woff) and np.array_equal(pos, wpos) and np.array_equal(slots, wslots)
    for i, s in enumerate(seqs):
        ids = [h[0] for h in cache.blocks(s)]
        assert tab[i].tolist() == ids + [-1] * (width - len(ids))


def test_slot_map_refusals_and_reports(device):
    say("slot map refusals")
    cache = device.PagedCache(1, 1, 2, 4, 16)
    a = cache.create_sequence()
    cache.reserve([a], [10])
    f = cache.fork(a)  # blocks 0..2 shared
    cache.reserve([f], [3])  # its tail block is its own now, as is the next one
    c = cache.create_sequence()
    seqs = [a, f, c]
    for starts, counts, stride, capacity in (([8, 10, 0], [2, 3, 0], 0, 16), ([0, 0, 0], [10, 13, 0], 0, 40),
                                             ([8, 10, 0], [2, 3, 1], 0, 16), ([8, -3, 0], [-5, 5, 0], 0, 16),
                                             ([10, 10, 0], [6, 3, 0], 0, 16), ([8, 10, 0], [2, 3, 0], 2, 6),
                                             ([8, 10, 0], [2, 3, 0], 0, 4), ([8, 10, 0], [2, 3, 0], 0, 0)):
        plan, off, pos, slots, _ = built(cache, seqs, starts, counts, stride, capacity, 0)
        woff, wpos, wslots, bad = plain_map(cache, seqs, starts, counts, stride, capacity)
        assert np.array_equal(off, woff) and np.array_equal(pos, wpos) and np.array_equal(slots, wslots), (starts, counts)
        if bad:
            with pytest.raises(_capi.InvalidArgument, match="slot map"):
                plan.check()
        plan.check()
    d = hip.DeviceArray.from_numpy(np.zeros(16, np.int32))
    for stride, capacity in ((3, 8), (1 << 40, 1 << 50)):
        with pytest.raises(_capi.InvalidArgument):
            plan.build(d.ptr, d.ptr, stride, capacity)
    with pytest.raises(_capi.InvalidArgument):
        plan.build(None, d.ptr, 0, 4)
    with pytest.raises(_capi.InvalidArgument):
        plan.build(d.ptr + 4, d.ptr, 0, 4)
    for bad in ([], [a, 99]):
        with pytest.raises(_capi.InvalidArgument):
            SlotPlan(cache, bad)
    cache.truncate(a, 3)
    with pytest.raises(_capi.InvalidArgument, match="stale"):
        plan.build(d.ptr, d.ptr, 0, 4)


def test_reserve(device):
    say("reserve")
    cache = device.PagedCache(2, 1, 4, 4, 8)
    a, b = cache.create_sequence(), cache.create_sequence()
    cache.append_many(a, np.ones((6, 8)), np.full((6, 8), 2.0))
    f = cache.fork(a)
    before = cache.state()
    with pytest.raises(_capi.CacheExhausted):
        cache.reserve([a, b], [3, 40])
    with pytest.raises(_capi.CacheExhausted):
        cache.reserve([a, b], [3, 17])
    with pytest.raises(_capi.CacheExhausted):  # each within the pool, together far beyond any memory
        cache.reserve([a] * 100000, [32] * 100000)
    with pytest.raises(_capi.CacheExhausted):
        cache.reserve([a, b], [1, (1 << 64) - 1])
    after = cache.state()
    assert {s: t[0] for s, t in after["tables"].items()} == {s: t[0] for s, t in before["tables"].items()}
    cache.audit()
    assert np.array_equal(cache.read_all(a, 0), np.ones(24)) and np.array_equal(cache.read_all(f, 1, True), np.full(24, 2.0))
    with pytest.raises(_capi.InvalidArgument):
        cache.reserve([a, 99], [1, 1])
    cache.reserve([a, f, a, b], [3, 0, 1, 5])
    assert cache.length(a) == 10 and cache.length(f) == 6 and cache.length(b) == 5
    cache.audit()
    assert np.array_equal(cache.read_all(a, 0)[:24], np.ones(24)) and not cache.read_all(b, 1).any()
    cache.reserve([], [])
    cache.reserve([a], [0])
    assert cache.length(a) == 10


@pytest.mark.parametrize("by_layer", [False, True])
@pytest.mark.parametrize("fmt,kv_heads,dim,tpb", [("f32", 2, 64, 16), ("f32", 8, 128, 16), ("f32", 1, 2, 3), ("f32", 3, 10, 4),
                                                  ("q8_0", 2, 64, 16), ("q8_0", 8, 128, 32), ("q8_0", 1, 32, 5)])
def test_slot_write(device, fmt, kv_heads, dim, tpb, by_layer):
    """The bytes that appends of the same rows leave; other slots keep theirs."""
    say("slot write", fmt, kv_heads, dim, tpb, by_layer)
    layers, w, n = 3, kv_heads * dim, 5
    r = np.random.default_rng(dim + tpb)
    f = device.Q8_0 if fmt == "q8_0" else device.F32
    caches = [device.PagedCache(layers, kv_heads, dim, tpb, 12 + 40 // tpb * n, fmt=f) for _ in range(2)]
    lengths, counts = [0, 1, tpb, 2 * tpb - 1, 7], [3, 0, 1, 4, 2]
    total = 20
    rows = r.normal(size=(2, total, layers, w)).astype(np.float32)
    rows[:, 3] = 0  # a group of zeros
    rows[0, 5, 0, 0] = 1e-42  # a subnormal scale
    pick = [np.sort(r.choice(total, c, replace=False)) for c in counts]
    pick[3][0] = 3
    seqs = []
    for cache in caches:
        mine = [cache.create_sequence() for _ in range(n)]
        for s, m in zip(mine, lengths):
            if m:
                old = np.full((m, layers * w), 0.5)
                cache.append_many(s, old, -old)
        seqs.append(mine)
    for s, p in zip(seqs[0], pick):
        if len(p):
            caches[0].append_many(s, rows[0, p], rows[1, p])
    cache = caches[1]
    cache.reserve(seqs[1], counts)
    up = hip.DeviceArray.from_numpy
    stride = max(counts) + 1
    plan = SlotPlan(cache, seqs[1])
    slots = hip.DeviceArray((n * stride,), np.int64)
    ds, dc = up(np.asarray(lengths, np.int32)), up(np.asarray(counts, np.int32))
    plan.build(ds.ptr, dc.ptr, stride, n * stride, slots_ptr=slots.ptr)
    chosen = np.full((n, stride), -1, np.int32)
    for i, p in enumerate(pick):
        chosen[i, :len(p)] = p
    dr = up(chosen)
    step = (w, total * w) if by_layer else (layers * w + 4, w)
    if by_layer:
        dk, dv = (up(np.ascontiguousarray(x.transpose(1, 0, 2))) for x in rows)
    else:
        dk, dv = (up(np.concatenate([x.reshape(total, -1), np.full((total, 4), np.nan, np.float32)], 1)) for x in rows)
    plan.write(slots.ptr, dr.ptr, n * stride, dk.ptr, dv.ptr, total, *step)
    plan.check()
    for s0, s1 in zip(*seqs):
        h0, h1 = caches[0].blocks(s0), cache.blocks(s1)
        assert caches[0].length(s0) == cache.length(s1) and len(h0) == len(h1)
        for x, y in zip(h0, h1):
            assert np.array_equal(caches[0].block_bytes_of(x), cache.block_bytes_of(y))


def test_slot_write_reports(device):
    say("slot write reports")
    cache = device.PagedCache(1, 1, 4, 4, 3)
    s = cache.create_sequence()
    cache.reserve([s], [12])
    up = hip.DeviceArray.from_numpy
    plan = SlotPlan(cache, [s])
    k, v = up(np.arange(16, dtype=np.float32).reshape(4, 4)), up(-np.arange(16, dtype=np.float32).reshape(4, 4))
    for slots, rows, bad in (([0, 11, -1], [0, 3, 9], False), ([12, 1], [0, 1], True), ([1 << 40, 1], [0, 1], True),
                             ([2, 1], [4, 1], True), ([2, 1], [-1, 1], True)):
        ds, dr = up(np.asarray(slots, np.int64)), up(np.asarray(rows, np.int32))
        plan.write(ds.ptr, dr.ptr, len(slots), k.ptr, v.ptr, 4, 4, 4)
        if bad:
            with pytest.raises(_capi.InvalidArgument, match="KV write"):
                plan.check()
        plan.check()
    got = cache.read_all(s, 0).reshape(12, 4)
    assert np.array_equal(got[0], np.arange(4)) and np.array_equal(got[11], np.arange(12, 16))
    assert np.array_equal(got[1], np.arange(4, 8)) and not got[2:11].any()
    ds = up(np.array([5, 6, 7, 8, 9], np.int64))
    plan.write(ds.ptr, None, 5, k.ptr, v.ptr, 4, 4, 4)  # row 4 of 4
    with pytest.raises(_capi.InvalidArgument):
        plan.check()
    assert np.array_equal(cache.read_all(s, 0).reshape(12, 4)[5:9], np.arange(16).reshape(4, 4))
    plan.write(None, None, 0, None, None, 0, 4, 4)
    for a in ((ds.ptr, None, 5, k.ptr, v.ptr, 4, 3, 4), (ds.ptr, None, 1 << 24, k.ptr, v.ptr, 4, 4, 4), (None, None, 5, k.ptr, v.ptr, 4, 4, 4),
              (ds.ptr, None, 5, k.ptr + 4, v.ptr, 4, 4, 4), (ds.ptr, None, 1 << 40, k.ptr, v.ptr, 4, 4, 4)):
        with pytest.raises(_capi.InvalidArgument):
            plan.write(*a)


# ------------------------------------------------------------ a whole step

class Graph:
    """A captured stream of launches, replayed."""

    def __init__(self, stream, body):
        self.rt = hip.runtime()
        self.stream = stream
        g, e = C.c_void_p(), C.c_void_p()
        hip.check(self.rt.hipStreamBeginCapture(C.c_void_p(stream), 2))  # relaxed
        try:
            body()
        finally:
            hip.check(self.rt.hipStreamEndCapture(C.c_void_p(stream), C.byref(g)))
        hip.check(self.rt.hipGraphInstantiate(C.byref(e), g, None, None, C.c_size_t(0)))
        self.g, self.e = g, e

    def replay(self):
        hip.check(self.rt.hipGraphLaunch(self.e, C.c_void_p(self.stream)))
        hip.check(self.rt.hipStreamSynchronize(C.c_void_p(self.stream)))

    def __del__(self):
        self.rt.hipGraphExecDestroy(self.e)
        self.rt.hipGraphDestroy(self.g)


class Step:
    """Buffers and plans of one speculative step of a Batch."""

    def __init__(self, b, vocab, seed, precision):
        r = np.random.default_rng(seed)
        self.b, self.vocab, self.depth = b, vocab, 8
        self.lengths = np.array(b.lengths, np.int32)
        b.cache.reserve(b.seqs, self.depth)
        up = hip.DeviceArray.from_numpy
        self.logits = r.normal(size=(b.rows, vocab)).astype(np.float32)
        at, self.tokens, self.first = 0, [], []
        for t in b.trees:
            mine = [int(r.integers(vocab)) if p < 0 or r.random() > 0.85 else int(np.argmax(self.logits[at + p]))
                    for p in t]
            self.tokens += mine
            self.first.append(mine[0] if mine else 0)
            at += len(t)
        n = len(b.trees)
        self.rows = r.normal(size=(2, b.rows, b.layers, b.w)).astype(np.float32)
        self.qs = r.normal(size=(b.layers, b.rows, b.heads * b.dim)).astype(np.float32)
        self.q, self.k, self.v = up(self.qs), up(self.rows[0]), up(self.rows[1])
        self.out = hip.DeviceArray(self.qs.shape)
        self.dl, self.dt, self.df = up(self.logits), up(np.array(self.tokens, np.uint32)), up(np.array(self.first, np.uint32))
        self.ds = up(self.lengths)
        self.path, self.acc = hip.DeviceArray((n, self.depth), np.int32), hip.DeviceArray((n,), np.int32)
        self.next, self.slots = hip.DeviceArray((n,), np.uint32), hip.DeviceArray((n * self.depth,), np.int64)
        self.slot_plan = SlotPlan(b.cache, b.seqs)
        self.plan = attention.TreePlan(b.cache, b.seqs, b.nodes, b.parents, b.heads, 1 << 20, visible=b.lengths,
                                       precision=precision)

    def launch(self, stream=None):
        b, step = self.b, self.b.layers * self.b.w
        for layer in range(b.layers):
            at = layer * b.w * 4
            self.plan.launch(layer, self.q.ptr + layer * b.rows * b.heads * b.dim * 4, self.k.ptr + at, self.v.ptr + at,
                             self.out.ptr + layer * b.rows * b.heads * b.dim * 4, row_stride=step, stream=stream)
        self.plan.accept(self.dt.ptr, self.df.ptr, self.dl.ptr, self.vocab, self.path.ptr, self.depth, self.acc.ptr,
                         self.next.ptr, stream=stream)
        n = len(b.trees)
        self.slot_plan.build(self.ds.ptr, self.acc.ptr, self.depth, n * self.depth, slots_ptr=self.slots.ptr, stream=stream)
        self.slot_plan.write(self.slots.ptr, self.path.ptr, n * self.depth, self.k.ptr, self.v.ptr, b.rows, step, b.w,
                             stream=stream)

    def verify(self, precision, finish=True):
        b = self.b
        self.plan.check()
        self.slot_plan.check()
        got, at = self.out.numpy(), 0
        for layer in range(b.layers):
            b.q, b.tk, b.tv = self.qs[layer], self.rows[0][:, layer], self.rows[1][:, layer]
            agree(got[layer], b.want(layer=layer), precision)
        acc, nxt = self.acc.numpy(), self.next.numpy()
        paths = []
        for i, t in enumerate(b.trees):
            want, after = walk(t, self.tokens[at:at + len(t)], self.first[i], self.logits[at:at + len(t)])
            assert len(want) <= self.depth and acc[i] == len(want) and nxt[i] == after
            paths.append([at + j for j in want])
            at += len(t)
        if finish:
            b.cache.truncate_batch(b.seqs, self.lengths + acc)
        for i, s in enumerate(b.seqs):
            for layer in range(b.layers):
                for kind, old in ((0, b.k[i]), (1, b.v[i])):
                    rows = b.cache.read_all(s, layer, bool(kind)).reshape(-1, b.w)[: self.lengths[i] + acc[i]]
                    new = self.rows[kind][paths[i], layer]
                    want = np.concatenate([old[:, layer * b.w:(layer + 1) * b.w], new])
                    if b.cache.format == _capi.KV_F32:
                        assert np.array_equal(rows, want.astype(np.float32))
                    else:  # half a step of the group's largest value
                        top = np.abs(want).reshape(-1, b.w // 32, 32).max(2).repeat(32, 1)
                        assert (np.abs(rows - want) <= top * (0.5 / 127 + 2.0 ** -11 + 1e-6)).all()
        b.cache.audit()


@pytest.mark.parametrize("precision", PRECISIONS)
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
def test_step(device, oracle, fmt, precision):
    say("tree step", fmt, precision)
    trees = [bushy(12, 3, 1, 0), bushy(7, 2, 2, 0), [], chain(6), bushy(20, 9, 3)]
    b = Batch(device, oracle, 8, 2, 64, [100, 33, 5, 0, 16], trees, layers=3, q8=fmt == "q8_0", seed=31, spare=8)
    step = Step(b, 500, 5, precision)
    step.launch()
    step.verify(precision)


def test_step_on_another_stream(device, oracle):
    """Everything on a stream of the caller's, the cache's own left on the null stream."""
    say("tree step, another stream")
    b = Batch(device, oracle, 8, 2, 128, [100, 333], [bushy(12, 3, 1, 0), bushy(7, 2, 2, 0)], layers=2, seed=32, spare=8)
    stream = hip.Stream()
    step = Step(b, 700, 6, "f32x3")
    step.launch(stream.h)
    step.verify("f32x3")


@pytest.mark.parametrize("precision", PRECISIONS)
def test_step_captured(device, oracle, precision):
    """A captured step, replayed with other work between, gives the eager bytes each time."""
    say("tree step captured", precision)
    b = Batch(device, oracle, 8, 2, 64, [1500, 33], [bushy(12, 3, 1, 0), bushy(7, 2, 2, 0)], layers=2, seed=33, spare=8)
    stream = hip.Stream()
    b.cache.set_stream(stream.h)
    step = Step(b, 300, 7, precision)
    step.launch(stream.h)
    hip.synchronize()
    eager = [x.numpy() for x in (step.out, step.path, step.acc, step.next, step.slots)]
    graph = Graph(stream.h, lambda: step.launch(stream.h))
    other = Batch(device, oracle, 8, 2, 64, [40], [chain(3)], seed=2)
    for _ in range(4):
        for x in (step.out, step.path, step.acc, step.next, step.slots):
            x.zero()
        hip.synchronize()
        graph.replay()
        for x, y in zip((step.out, step.path, step.acc, step.next, step.slots), eager):
            assert np.array_equal(x.numpy(), y)
        agree(other.run(), other.want(), "f32")
    step.verify(precision)
    del graph
    b.cache.set_stream(None)


def test_two_plans_on_two_streams(device, oracle):
    """Two plans' launches at once share nothing."""
    say("two tree plans at once")
    bs = [Batch(device, oracle, 8, 2, 64, [900, 400], [bushy(9, 3, i), chain(5)], seed=40 + i) for i in range(2)]
    streams = [hip.Stream() for _ in bs]
    ds = [hip_rows(b) for b in bs]
    plans = [attention.TreePlan(b.cache, b.seqs, b.nodes, b.parents, b.heads, 1 << 20) for b in bs]
    for _ in range(5):
        for p, d, s in zip(plans, ds, streams):
            p.launch(0, d.q.ptr, d.k.ptr, d.v.ptr, d.out.ptr, stream=s.h)
    for p, d, b in zip(plans, ds, bs):
        p.check()
        agree(d.out.numpy()[: b.rows], b.want(), "f32")
