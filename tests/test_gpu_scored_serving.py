"""Scored attention, rotation into the cache, reading back and sampling as a server runs
them: two layers with capped scores, a bias by distance and a window take a ragged batch
from their fused rows to the drawn tokens, the same step captured and replayed.

Each link is held to its own bar, on what the link before it left: cached keys to u =
2^-24 of themselves and 2^-40 of their pair (Q8_0: to half a step of amax / 127, and the
scale's rounding to fp16, 127 x 2^-11 of a step), attention to the formula over the
cache's rows as in test_gpu_score (and one u more of a score for the query's rounding),
tokens to numpy's draw from the same logits as in test_gpu_sample.
"""

import sys

import numpy as np
import pytest

import test_gpu_sample as ts
import test_gpu_tree as tt
from tvara_amd import attention, hip, synth
from tvara_amd.kv import SlotPlan
from tvara_amd.sampling import SamplePlan

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
LAYERS, HEADS, KV, DIM, TPB, VOCAB, WINDOW, CAP, BASE = 2, 8, 2, 64, 16, 5000, 40, 20.0, 10000.0
HIDDEN, WIDTH = HEADS * DIM, KV * DIM
FREQS = (BASE ** (-np.arange(DIM // 2) / (DIM // 2))).astype(np.float32)
SLOPES = (2.0 ** -np.arange(1, HEADS + 1)).astype(np.float32)


def say(*a):
    print(*a, flush=True, file=sys.stderr)


def upload(device_array, values):
    values = np.ascontiguousarray(values, device_array.dtype)
    hip.check(hip.runtime().hipMemcpy(device_array.ptr, values.ctypes.data, values.nbytes, hip.H2D))


def rotated(x, positions, weight):
    """In 64 bits, and each element's pair's size."""
    x = x.astype(np.float64)
    x = x / np.sqrt((x * x).mean(2, keepdims=True) + 1e-6) * weight.astype(np.float64)
    t = positions.astype(np.float64)[:, None, None] * FREQS.astype(np.float64)
    a, b = x[..., : DIM // 2], x[..., DIM // 2:]
    y = np.concatenate([a * np.cos(t) - b * np.sin(t), a * np.sin(t) + b * np.cos(t)], 2)
    return y, np.concatenate([np.hypot(a, b)] * 2, 2)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("counts", [[1, 1, 1], [5, 1, 90]])
def test_layers_to_tokens(device, q8, counts):
    say("scored serving", q8, counts)
    rng = np.random.default_rng(sum(counts) + q8)
    lengths, n, rows = [17, 0, 120], len(counts), sum(counts)
    cache = device.PagedCache(LAYERS, KV, DIM, TPB, 64, fmt=device.Q8_0 if q8 else device.F32)
    seqs = []
    for i, length in enumerate(lengths):
        seqs.append(cache.create_sequence())
        if length:
            cache.append_many(seqs[-1], *(synth.normal(5, f"{x}{i}", length * LAYERS * WIDTH).reshape(length, -1) for x in "kv"))
    cache.reserve(seqs, counts)
    first, end = attention.visible_ranges(lengths, counts, window=WINDOW)
    positions = np.concatenate([s + np.arange(c) for s, c in zip(lengths, counts)])
    slots, sampled = SlotPlan(cache, seqs), SamplePlan(n, VOCAB)
    scored = attention.ScorePlan(cache, seqs, lengths, counts, HEADS, 1 << 16, first, end, cap=CAP, slopes=SLOPES)
    up = hip.DeviceArray.from_numpy
    wq, wk = ((1 + 0.2 * rng.normal(size=DIM)).astype(np.float32) for _ in "qk")
    head = (rng.normal(size=(HIDDEN, VOCAB)) / 4).astype(np.float32)
    dq, dk, freqs = up(wq), up(wk), up(FREQS)
    dstarts, dcounts = up(np.array(lengths, np.int32)), up(np.array(counts, np.int32))
    pos, slot_ids = hip.DeviceArray((rows,), np.int32), hip.DeviceArray((rows,), np.int64)
    fused = [hip.DeviceArray((rows, HIDDEN + 2 * WIDTH)) for _ in range(LAYERS)]
    queries, outs = hip.DeviceArray((rows, HIDDEN)), [hip.DeviceArray((rows, HIDDEN)) for _ in range(LAYERS)]
    back = [hip.DeviceArray((rows, LAYERS * WIDTH)) for _ in "kv"]
    logits, uniforms = hip.DeviceArray((n, VOCAB)), hip.DeviceArray((n,))
    tokens, chances = hip.DeviceArray((n,), np.uint32), hip.DeviceArray((n,))
    params = [up(np.full(n, v, t)) for v, t in ((0.8, np.float32), (200, np.int32), (0.95, np.float32), (1e-3, np.float32))]
    stream = hip.Stream()
    hip.synchronize()

    def layers():
        slots.build(dstarts.ptr, dcounts.ptr, 0, rows, None, pos.ptr, slot_ids.ptr, stream=stream.h)
        for layer in range(LAYERS):
            p, stride = fused[layer].ptr, HIDDEN + 2 * WIDTH
            slots.rotate(slot_ids.ptr, rows, layer, p, p + 4 * HIDDEN, p + 4 * (HIDDEN + WIDTH), pos.ptr, freqs.ptr, DIM, HEADS,
                         queries.ptr, None, stride, stride, dq.ptr, dk.ptr, 1e-6, stream=stream.h)
            scored.launch(layer, queries.ptr, outs[layer].ptr, stream=stream.h)
        slots.read(slot_ids.ptr, rows, 0, LAYERS, back[0].ptr, back[1].ptr, LAYERS * WIDTH, WIDTH, stream=stream.h)

    def draw():
        sampled.launch(logits.ptr, uniforms.ptr, tokens.ptr, chances.ptr, *(p.ptr for p in params), stream=stream.h)

    def check_layer(layer, x):
        q, k, v = np.split(x, [HIDDEN, HIDDEN + WIDTH], 1)
        q, _ = rotated(q.reshape(rows, HEADS, DIM), positions, wq)
        k, size = (y.reshape(rows, WIDTH) for y in rotated(k.reshape(rows, KV, DIM), positions, wk))
        want, bar = np.zeros((2, rows, HEADS, DIM))
        r = 0
        for i, c in enumerate(counts):
            kk, vv = (cache.read_all(seqs[i], layer, value).astype(np.float64).reshape(-1, WIDTH) for value in (False, True))
            for value, (held, given) in enumerate(((kk, k), (vv, v.astype(np.float64)))):
                new, given = held[lengths[i]:], given[r: r + c]
                if q8:
                    step = abs(given.reshape(c, -1, 32)).max(2, keepdims=True) / 127
                    off = np.broadcast_to((0.5 + 127 * 2.0 ** -11) * (1 + 2.0 ** -10) * step, (c, WIDTH // 32, 32)).reshape(c, -1)
                else:
                    off = 0 if value else U * abs(given) + 2.0 ** -40 * size[r: r + c]
                assert (abs(new - given) <= off).all()
                cols = slice(layer * WIDTH, (layer + 1) * WIDTH)
                assert np.array_equal(back[value].numpy()[r: r + c, cols], new)
            kk, vv = (np.repeat(y.reshape(-1, KV, DIM), HEADS // KV, 1).transpose(1, 0, 2) for y in (kk, vv))
            for j in range(r, r + c):
                seen = slice(int(first[j]), int(end[j]))
                a, b = kk[:, seen], vv[:, seen]
                s = (q[j][:, None] * a).sum(2) / np.sqrt(DIM)
                e = (DIM + 9) * U * (abs(q[j][:, None]) * abs(a)).sum(2) / np.sqrt(DIM) + 8 * U * CAP
                s = CAP * np.tanh(s / CAP)
                away = SLOPES.astype(np.float64)[:, None] * abs(positions[j] - np.arange(seen.start, seen.stop))
                s, e = s - away, e + 2 * U * away + U * abs(s - away)
                w = np.exp(s - s.max(1, keepdims=True))
                w /= w.sum(1, keepdims=True)
                want[j] = (w[:, :, None] * b).sum(1)
                bar[j] = (2 * e.max(1) + (16 + (seen.stop - seen.start) / 32 + 64) * U)[:, None] * (w[:, :, None] * abs(b)).sum(1)
            r += c
        assert (abs(outs[layer].numpy() - want.reshape(rows, -1)) <= bar.reshape(rows, -1)).all()

    def step(run_layers, run_draw):
        given = [rng.normal(size=(rows, HIDDEN + 2 * WIDTH)).astype(np.float32) for _ in range(LAYERS)]
        for d, x in zip(fused, given):
            upload(d, x)
        for d in outs + back + [tokens, chances]:
            d.zero()
        hip.synchronize()
        run_layers()
        scored.check()
        slots.check()
        for layer, x in enumerate(given):
            check_layer(layer, x)
        # (the product with the head is the host's here)
        x, u = outs[-1].numpy()[np.cumsum(counts) - 1] @ head, rng.random(n).astype(np.float32)
        upload(logits, x)
        upload(uniforms, u)
        hip.synchronize()
        run_draw()
        sampled.check()
        for i in range(n):
            token, chance = ts.draw(x[i], u[i], 0.8, 200, 0.95, 1e-3)
            assert tokens.numpy()[i] == token
            assert abs(chances.numpy()[i] - chance) <= (U + 1e-9) * chance

    step(layers, draw)
    cache.set_stream(stream.h)
    graphs = [tt.Graph(stream.h, f) for f in (layers, draw)]
    for _ in range(3):
        step(graphs[0].replay, graphs[1].replay)
    del graphs
    hip.synchronize()
    cache.set_stream(None)
