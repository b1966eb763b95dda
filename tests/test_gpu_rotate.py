"""Rows into the cache and out of it on the GPU: queries and keys normalised and
rotated, written into slots as f32 or Q8_0, and read back.

The arithmetic is in f64 and rounded once, so an output is off by u = 2^-24 of itself
for the rounding and by a few 2^-53 of its pair's size for the rest: the bar is u |y| +
2^-45 |pair|.  Angles: position * freq is one rounding of f64, 2^-53 * 2^31 / 2 at the
most, which the formula's has too.  A Q8_0 byte and scale are those of the rounded f32
value; that value may differ by one unit where it falls within 2^-45 of a border, which
no seed here does, so bytes are equal.
"""

import sys

import numpy as np
import pytest

import test_gpu_tree as tt
from tvara_amd import _capi, attention, hip, synth
from tvara_amd.kv import SlotPlan

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def say(*a):
    print(*a, flush=True, file=sys.stderr)


def turned(x, positions, freqs, rotary, interleaved, weight, eps):
    """x [n, heads, dim] in 64 bits, and the size of each element's pair."""
    x = x.astype(np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(2, keepdims=True) + eps) * weight.astype(np.float64)
    y, size = x.copy(), abs(x)
    t = positions.astype(np.float64)[:, None, None] * freqs.astype(np.float64)
    a = np.arange(0, rotary, 2) if interleaved else np.arange(rotary // 2)
    b = a + 1 if interleaved else a + rotary // 2
    y[..., a] = x[..., a] * np.cos(t) - x[..., b] * np.sin(t)
    y[..., b] = x[..., a] * np.sin(t) + x[..., b] * np.cos(t)
    size[..., a] = size[..., b] = np.hypot(x[..., a], x[..., b])
    return y, U * abs(y) + 2.0 ** -45 * size


class Rows:
    """A layer's fused rows for n tokens, with a cache that has a slot for each."""

    def __init__(self, device, heads, kv_heads, dim, n, tpb=16, q8=False, layers=2, fused=True, seed=3, far=5000, extra=0):
        self.heads, self.kv_heads, self.dim, self.n, self.q8 = heads, kv_heads, dim, n, q8
        self.hidden, self.w = heads * dim, kv_heads * dim
        r = np.random.default_rng(seed + n + dim)
        width = self.hidden + 2 * self.w + extra
        self.x = r.normal(size=(n, width)).astype(np.float32)
        self.q, self.k, self.v = np.split(self.x[:, : self.hidden + 2 * self.w], [self.hidden, self.hidden + self.w], 1)
        self.pos = r.integers(0, far, n).astype(np.int32)
        blocks = -(-n // tpb) + 1
        self.cache = device.PagedCache(layers, kv_heads, dim, tpb, blocks, fmt=device.Q8_0 if q8 else device.F32)
        self.seq = self.cache.create_sequence()
        self.cache.reserve([self.seq], [blocks * tpb])
        self.slots = r.permutation(blocks * tpb)[:n].astype(np.int64)
        order = [b for b, _ in self.cache.blocks(self.seq)]
        where = {b * tpb + i: o * tpb + i for o, b in enumerate(order) for i in range(tpb)}
        self.at = np.array([where[int(s)] for s in self.slots])  # each slot's place in the sequence
        up = hip.DeviceArray.from_numpy
        if fused:
            d = up(self.x)
            self.ptrs = [d.ptr, d.ptr + 4 * self.hidden, d.ptr + 4 * (self.hidden + self.w)]
            self.strides = {"q_stride": width, "kv_stride": width}
            self.dev = [d]
        else:
            self.dev = [up(np.ascontiguousarray(y)) for y in (self.q, self.k, self.v)]
            self.ptrs, self.strides = [d.ptr for d in self.dev], {}
        self.plan = SlotPlan(self.cache, [self.seq])
        self.freqs = (10000.0 ** (-np.arange(dim // 2) / (dim // 2))).astype(np.float32)
        self.wq, self.wk = (1 + 0.3 * r.normal(size=dim)).astype(np.float32), (1 + 0.3 * r.normal(size=dim)).astype(np.float32)

    def run(self, rotary, interleaved, norm, layer=1, slots=None, k_out=False, q_out=True, stream=None):
        up = hip.DeviceArray.from_numpy
        self.keep = [up(self.slots if slots is None else slots), up(self.pos), up(self.freqs), up(self.wq), up(self.wk)]
        s, p, f, wq, wk = (d.ptr for d in self.keep)
        self.q_out = hip.DeviceArray((self.n, self.hidden)) if q_out else None
        self.k_out = hip.DeviceArray((self.n, self.w)) if k_out else None
        how = {"q_norm_ptr": wq, "k_norm_ptr": wk, "eps": 1e-5} if norm else {}
        self.plan.rotate(s, self.n, layer, *self.ptrs, p, f, rotary, self.heads, self.q_out and self.q_out.ptr,
                         self.k_out and self.k_out.ptr, interleaved=interleaved, stream=stream, **how, **self.strides)
        self.plan.check()

    def want(self, rotary, interleaved, norm):
        f = self.freqs[: rotary // 2]
        out = []
        for x, w in ((self.q, self.wq), (self.k, self.wk)):
            y, bar = turned(x.reshape(self.n, -1, self.dim), self.pos, f, rotary, interleaved, w if norm else None, 1e-5)
            out.append((y.reshape(self.n, -1), bar.reshape(self.n, -1)))
        return out

    def cached(self, layer):
        return [self.cache.read_all(self.seq, layer, value).reshape(-1, self.w) for value in (False, True)]

    def agree(self, oracle, rotary, interleaved, norm, layer=1, live=None):
        (q, q_bar), (k, k_bar) = self.want(rotary, interleaved, norm)
        if self.q_out:
            assert (abs(self.q_out.numpy() - q) <= q_bar).all()
        if self.k_out:
            assert (abs(self.k_out.numpy() - k) <= k_bar).all()
        live = np.ones(self.n, bool) if live is None else live
        keys, values = self.cached(layer)
        at = self.at[live]
        if self.q8:
            held = [oracle.dequantize_q8_0(oracle.quantize_q8_0(np.ascontiguousarray(y[live], np.float32))).reshape(-1, self.w)
                    for y in (k, self.v)]
            assert np.array_equal(keys[at], held[0]) and np.array_equal(values[at], held[1])
        else:
            assert (abs(keys[at] - k[live]) <= k_bar[live]).all()
            assert np.array_equal(values[at], self.v[live])
        rest = np.ones(len(keys), bool)
        rest[at] = False
        assert not keys[rest].any() and not values[rest].any()
        for other in range(self.cache.layers):
            if other != layer:
                assert not any(x.any() for x in self.cached(other))


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
@pytest.mark.parametrize("heads,kv_heads,dim,rotary", [(9, 3, 64, 64), (4, 2, 128, 128), (4, 2, 128, 64), (3, 1, 64, 32), (2, 1, 256, 256),
                                                       (6, 2, 96, 96), (2, 2, 32, 8), (4, 2, 64, 36), (2, 1, 160, 40), (2, 1, 64, 0)])
def test_rotate(device, oracle, heads, kv_heads, dim, rotary, fmt, interleaved, norm):
    say("rotate", heads, kv_heads, dim, rotary, fmt, interleaved, norm)
    b = Rows(device, heads, kv_heads, dim, 21, q8=fmt == "q8_0")
    b.run(rotary, interleaved, norm, k_out=True)
    b.agree(oracle, rotary, interleaved, norm)


@pytest.mark.parametrize("dim,tpb", [(8, 3), (16, 16), (512, 1), (6, 5), (10, 16)])
def test_head_sizes_of_f32_blocks(device, oracle, dim, tpb):
    say("rotate, head sizes", dim, tpb)
    b = Rows(device, 4, 2, dim, 7, tpb=tpb)
    b.run(dim - dim % 4, False, True)
    b.agree(oracle, dim - dim % 4, False, True)


@pytest.mark.parametrize("n", [1, 2, 63, 1023, 1024, 2100])
@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
def test_counts(device, oracle, fmt, n):
    """One token to a prompt's; every eighth has no slot, and its queries all the same."""
    say("rotate, counts", fmt, n)
    b = Rows(device, 9, 3, 64, n, q8=fmt == "q8_0", far=1 << 20)
    slots, live = b.slots.copy(), np.arange(n) % 8 != 7
    slots[~live] = -1
    b.run(64, False, True, slots=slots)
    b.agree(oracle, 64, False, True, live=live)


@pytest.mark.parametrize("extra", [0, 1, 4])
@pytest.mark.parametrize("fused", [True, False])
def test_strides(device, oracle, fused, extra):
    """Rows of a fused product, packed rows, and rows whose stride is no multiple of 4."""
    say("rotate, strides", fused, extra)
    b = Rows(device, 4, 2, 64, 9, fused=fused, extra=extra if fused else 0, layers=1)
    b.run(64, True, True, layer=0)
    b.agree(oracle, 64, True, True, layer=0)


def test_far_positions_and_large_frequencies(device, oracle):
    say("rotate, far")
    b = Rows(device, 4, 2, 64, 8)
    b.pos = np.array([0, 1, 2**20 + 1, 2**24 + 3, 2**30 + 7, 2**31 - 1, -1, -(2**31)], np.int32)
    b.freqs[:4] = 1.0, 3.14159274, 0.5, 7.25
    b.run(64, False, False)
    (q, bar), _ = b.want(64, False, False)
    # 2^31 * 7.25 is 2^34: a rounding of the product is 2^-19 of a radian, the same in both
    assert (abs(b.q_out.numpy() - q) <= bar + 2.0 ** -45 * abs(q)).all()


def test_queries_in_place_and_only_what_is_asked(device, oracle):
    say("rotate, parts")
    b = Rows(device, 4, 2, 64, 5, fused=False)
    up = hip.DeviceArray.from_numpy
    pos, freqs = up(b.pos), up(b.freqs)
    (q, q_bar), (k, k_bar) = b.want(64, False, False)
    # queries alone, onto themselves
    b.plan.rotate(None, 5, 0, b.ptrs[0], None, None, pos.ptr, freqs.ptr, 64, 4, b.ptrs[0])
    # keys alone, to rows
    keys = hip.DeviceArray((5, b.w))
    b.plan.rotate(None, 5, 0, None, b.ptrs[1], None, pos.ptr, freqs.ptr, 64, 4, None, keys.ptr)
    b.plan.check()
    assert (abs(b.dev[0].numpy() - q) <= q_bar).all() and (abs(keys.numpy() - k) <= k_bar).all()
    assert not any(x.any() for x in b.cached(0))
    b.plan.rotate(None, 0, 0, None, None, None, None, None, 64, 4, None)


@pytest.mark.parametrize("fmt", ["f32", "q8_0"])
@pytest.mark.parametrize("kv_heads,dim", [(3, 64), (2, 128), (1, 96), (2, 10)])
@pytest.mark.parametrize("layer,layers", [(0, 3), (1, 1), (2, 1), (1, 2), (1, 0)])
def test_read(device, oracle, layer, layers, kv_heads, dim, fmt):
    if fmt == "q8_0" and dim % 32:
        return
    say("read", layer, layers, kv_heads, dim, fmt)
    b = Rows(device, kv_heads, kv_heads, dim, 37, q8=fmt == "q8_0", layers=3)
    up = hip.DeviceArray.from_numpy
    rows = [synth.normal(5, x, b.n * 3 * b.w).reshape(b.n, 3, b.w) for x in "kv"]
    given = [up(x) for x in rows]
    slots = b.slots.copy()
    all_slots = up(slots)
    b.plan.write(all_slots.ptr, None, b.n, given[0].ptr, given[1].ptr, b.n, 3 * b.w, b.w)
    slots[::5] = -1
    some = up(slots)
    for by_layer in (False, True):
        shape = (max(layers, 1), b.n, b.w) if by_layer else (b.n, max(layers, 1), b.w)
        outs = [up(np.full(shape, 7.5, np.float32)) for _ in "kv"]
        strides = (b.w, b.n * b.w) if by_layer else (max(layers, 1) * b.w, b.w)
        b.plan.read(some.ptr, b.n, layer, layers, outs[0].ptr, outs[1].ptr, *strides)
        b.plan.check()
        for x, o in zip(rows, outs):
            if b.q8:
                x = oracle.dequantize_q8_0(oracle.quantize_q8_0(np.ascontiguousarray(x))).reshape(x.shape)
            want = np.full((b.n, max(layers, 1), b.w), 7.5, np.float32)
            want[slots >= 0, :layers] = x[slots >= 0, layer : layer + layers]
            assert np.array_equal(o.numpy(), want.transpose(1, 0, 2) if by_layer else want)


def test_bad_slots_are_reported(device, oracle):
    say("rotate and read, bad slots")
    b = Rows(device, 4, 2, 64, 6)
    slots, end = b.slots.copy(), b.cache.max_blocks * 16
    slots[2], slots[4] = end, -7  # (below zero: none)
    with pytest.raises(_capi.InvalidArgument, match="outside the pool"):
        b.run(64, False, False, slots=slots)
    live = np.array([1, 1, 0, 1, 0, 1], bool)
    b.agree(oracle, 64, False, False, live=live)
    up = hip.DeviceArray.from_numpy
    s, outs = up(slots), [up(np.full((6, b.w), 2.0, np.float32)) for _ in "kv"]
    b.plan.read(s.ptr, 6, 1, 1, outs[0].ptr, outs[1].ptr, b.w, 0)
    with pytest.raises(_capi.InvalidArgument, match="outside the pool"):
        b.plan.check()
    keys, _ = b.cached(1)
    assert np.array_equal(outs[0].numpy()[live], keys[b.at[live]]) and (outs[0].numpy()[~live] == 2).all()
    b.plan.check()


def test_refusals(device, oracle):
    say("rotate and read, refusals")
    b = Rows(device, 4, 2, 64, 4)
    up = hip.DeviceArray.from_numpy
    d = up(np.zeros(4096, np.float32))
    s = up(b.slots)
    bad = _capi.InvalidArgument

    def rotate(slots=s.ptr, n=4, layer=0, q=d.ptr, k=d.ptr, v=d.ptr, pos=d.ptr, freqs=d.ptr, rotary=64, heads=4, q_out=d.ptr, **how):
        b.plan.rotate(slots, n, layer, q, k, v, pos, freqs, rotary, heads, q_out, **how)

    for how in ({"layer": 2}, {"layer": 1 << 40}, {"heads": 3}, {"heads": 0}, {"heads": 1 << 33}, {"rotary": 66}, {"rotary": 3},
                {"q": None}, {"k": None}, {"v": None}, {"pos": None}, {"freqs": None}, {"q": d.ptr + 4}, {"slots": s.ptr + 8},
                {"q_out": d.ptr + 8}, {"eps": -1.0}, {"eps": np.nan}, {"q_stride": 255}, {"kv_stride": 127}, {"n": 1 << 40},
                {"q_norm_ptr": d.ptr + 4}, {"k_out_ptr": d.ptr + 4}):
        with pytest.raises(bad):
            rotate(**how)

    def read(slots=s.ptr, n=4, layer=0, layers=1, k=d.ptr, v=d.ptr, row=128, lay=0):
        b.plan.read(slots, n, layer, layers, k, v, row, lay)

    for how in ({"layer": 2}, {"layers": 3}, {"layer": 1, "layers": 2, "lay": 128}, {"slots": None}, {"k": None}, {"v": None},
                {"k": d.ptr + 4}, {"row": 127}, {"layers": 2, "lay": 100}, {"n": 1 << 40}, {"layer": 1 << 40}):
        with pytest.raises(bad):
            read(**how)
    b.cache.truncate(b.seq, 3)
    with pytest.raises(bad, match="stale"):
        rotate()
    with pytest.raises(bad, match="stale"):
        read()


def test_captured_and_on_another_stream(device, oracle):
    say("rotate, captured")
    b = Rows(device, 4, 2, 64, 40, q8=True)
    stream = hip.Stream()
    hip.synchronize()
    b.run(64, False, True, stream=stream.h)
    b.agree(oracle, 64, False, True)
    eager = b.q_out.numpy()
    b.cache.set_stream(stream.h)
    s, p, f, wq, wk = (d.ptr for d in b.keep)
    outs = [hip.DeviceArray((b.n, b.w)) for _ in "kv"]

    def both():
        b.plan.rotate(s, b.n, 1, *b.ptrs, p, f, 64, 4, b.q_out.ptr, q_norm_ptr=wq, k_norm_ptr=wk, eps=1e-5, stream=stream.h, **b.strides)
        b.plan.read(s, b.n, 1, 1, outs[0].ptr, outs[1].ptr, b.w, 0, stream=stream.h)

    graph = tt.Graph(stream.h, both)
    for _ in range(3):
        b.q_out.zero()
        outs[0].zero()
        hip.synchronize()
        graph.replay()
        b.plan.check()
        assert np.array_equal(b.q_out.numpy(), eager)
        assert np.array_equal(outs[0].numpy(), b.cached(1)[0][b.at])
    del graph
    hip.synchronize()
    b.cache.set_stream(None)


@pytest.mark.parametrize("dim,interleaved,norm", [(64, False, True), (128, True, True), (10, False, True), (20, True, False)])
def test_in_place(device, oracle, dim, interleaved, norm):
    """Packed queries and keys onto themselves, in the kernel of eight columns a thread and in
    the other; rows with something between them are refused."""
    say("rotate, in place", dim, interleaved, norm)
    b = Rows(device, 4, 2, dim, 9, fused=False)
    up = hip.DeviceArray.from_numpy
    pos, freqs, wq, wk = up(b.pos), up(b.freqs), up(b.wq), up(b.wk)
    how = {"q_norm_ptr": wq.ptr, "k_norm_ptr": wk.ptr, "eps": 1e-5} if norm else {}
    call = [b.ptrs[0], b.ptrs[1], None, pos.ptr, freqs.ptr, dim, 4, b.ptrs[0], b.ptrs[1]]
    for strides in ({"q_stride": 4 * dim + 4}, {"kv_stride": 2 * dim + 4}):
        with pytest.raises(_capi.InvalidArgument, match="overlap"):
            b.plan.rotate(None, 9, 0, *call, interleaved=interleaved, **how, **strides)
    b.plan.rotate(None, 9, 0, *call, interleaved=interleaved, **how)
    b.plan.check()
    for got, (want, bar) in zip(b.dev, b.want(dim, interleaved, norm)):
        assert (abs(got.numpy() - want) <= bar).all()


def test_rows_read_over_each_other_are_refused(device, oracle):
    say("read, overlapping rows")
    b = Rows(device, 4, 2, 64, 4, layers=3)
    d, s, w = hip.DeviceArray((4 * 3 * 128 + 8,)), hip.DeviceArray.from_numpy(b.slots), 128
    for row, layer in ((w, w), (2 * w, w), (3 * w - 4, w), (w, 4 * w - 4), (1 << 62, 1 << 61)):
        with pytest.raises(_capi.InvalidArgument, match="overlap"):
            b.plan.read(s.ptr, 4, 0, 3, d.ptr, d.ptr, row, layer)
    for n, layers, row, layer in ((4, 3, 3 * w, w), (4, 3, w, 4 * w), (1, 3, w, w), (4, 1, w, 0)):
        b.plan.read(s.ptr, n, 0, layers, d.ptr, d.ptr, row, layer)
    b.plan.check()


def test_rows_that_pass_the_address_space_are_refused(device, oracle):
    say("rotate, strides without end")
    b = Rows(device, 4, 2, 64, 4)
    d, s = hip.DeviceArray.from_numpy(np.zeros(4096, np.float32)), hip.DeviceArray.from_numpy(b.slots)
    for how in ({"q_stride": 1 << 62}, {"kv_stride": 1 << 62}, {"q_stride": 1 << 58}, {"kv_stride": (1 << 64) - 4}):
        with pytest.raises(_capi.InvalidArgument, match="overlap"):
            b.plan.rotate(s.ptr, 4, 0, d.ptr, d.ptr, d.ptr, d.ptr, d.ptr, 64, 4, None, **how)
    for n, row, layer in ((4, 1 << 62, 0), (1, 128, 1 << 62), (4, (1 << 64) - 4, 128)):
        with pytest.raises(_capi.InvalidArgument, match="overlap"):
            b.plan.read(s.ptr, n, 0, 2, d.ptr, d.ptr, row, layer)
    b.plan.check()
