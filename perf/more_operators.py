"""What one decode or prompt step of a served model is timed on beyond plain
attention: queries and keys normalised, rotated and written into the paged
cache, attention with capped or biased scores over what each row may see, rows
read back from the cache, and the choice of the next token.

``listed()`` names the cases and ``draw()`` gives others of the same ranges.  A
case is a plain dict; lengths, visible ranges and block orders follow from its
own fields, every value that is computed on from the seed.  Four kinds:

score    one ``ScorePlan.launch``: rows of queries over their sequences' cached
         tokens, each within a range of its own.
rotate   one ``SlotPlan.rotate`` of a layer, with ``SlotPlan.read`` behind it
         over quantised blocks.
read     one ``SlotPlan.read``: K and V rows of several layers out of slots.
sample   one ``SamplePlan.launch``: a batch's next tokens from given random numbers.

``own`` says whether ``run`` calls the framework or computes in plain torch.
The framework's cache keeps its blocks itself, so only its side fills one.
"""

import math
import random
import zlib

import numpy as np
import torch

own = False

CONTEXT = 1 << 20
DEVICE = "cuda"

# (query heads, KV heads, head_dim) of the attention layers in use here:
# SmolLM2-135M, Llama-3.2-1B, Llama-3-8B, Llama-3-70B, TinyLlama-1.1B
SMOL, L1B, L8B, L70B, TINY = (9, 3, 64), (32, 8, 64), (32, 8, 128), (64, 8, 128), (32, 4, 64)


def _shape(s):
    return {"heads": s[0], "kv_heads": s[1], "dim": s[2]}


def listed():
    return [
        # one user's stream on a small model, capped scores: launch-bound
        {"name": "score-smol-1x700-cap", "kind": "score", **_shape(SMOL), "n": 1, "low": 700, "high": 700, "rlow": 1,
         "rhigh": 1, "cap": 30.0, "slopes": False, "window": 0, "prefix": 0, "document": 0, "block": 16, "q8": False,
         "spread": 1},
        # a serving batch of unequal contexts, a bias by distance
        {"name": "score-1b-48-slopes", "kind": "score", **_shape(L1B), "n": 48, "low": 100, "high": 3000, "rlow": 1,
         "rhigh": 1, "cap": 0.0, "slopes": True, "window": 0, "prefix": 0, "document": 0, "block": 16, "q8": False,
         "spread": 2},
        # few long contexts over quantised blocks of 64 tokens
        {"name": "score-8b-q8-8x32k-cap", "kind": "score", **_shape(L8B), "n": 8, "low": 16000, "high": 32768,
         "rlow": 1, "rhigh": 1, "cap": 50.0, "slopes": False, "window": 0, "prefix": 0, "document": 0, "block": 64,
         "q8": True, "spread": 3},
        # two prompts' second chunks: the most arithmetic
        {"name": "score-8b-prompt-2x2048-cap", "kind": "score", **_shape(L8B), "n": 2, "low": 4096, "high": 4096,
         "rlow": 2048, "rhigh": 2048, "cap": 50.0, "slopes": False, "window": 0, "prefix": 0, "document": 0,
         "block": 16, "q8": False, "spread": 4},
        # ragged prompts in one batch, a window behind a common prefix
        {"name": "score-1b-prompts-window", "kind": "score", **_shape(L1B), "n": 6, "low": 700, "high": 2500,
         "rlow": 3, "rhigh": 700, "cap": 0.0, "slopes": True, "window": 600, "prefix": 150, "document": 0,
         "block": 32, "q8": False, "spread": 5},
        # one user's token
        {"name": "rotate-smol-1", "kind": "rotate", **_shape(SMOL), "n": 1, "norm": False, "interleaved": True,
         "rotary": 64, "block": 16, "q8": False, "far": 600, "spread": 6},
        # a serving batch with normalised queries and keys, quantised as they are written and read back
        {"name": "rotate-8b-64-q8-read", "kind": "rotate", **_shape(L8B), "n": 64, "norm": True, "interleaved": False,
         "rotary": 128, "block": 16, "q8": True, "far": 32768, "spread": 7},
        # a prompt pass's tokens
        {"name": "rotate-8b-4000", "kind": "rotate", **_shape(L8B), "n": 4000, "norm": True, "interleaved": False,
         "rotary": 128, "block": 16, "q8": False, "far": 131072, "spread": 8},
        # a text's rows of four layers, to be kept elsewhere
        {"name": "read-8b-q8-1500x4-layers", "kind": "read", **_shape(L8B), "n": 1500, "layers": 4, "block": 64,
         "q8": True, "spread": 9},
        # one user's next token
        {"name": "sample-32k-1", "kind": "sample", "n": 1, "vocab": 32000, "temperature": 0.8, "top_k": 50,
         "top_p": 0.95, "min_p": 0.0, "mixed": False, "bulk": 2.0, "spread": 10},
        # a batch whose requests ask for different things
        {"name": "sample-128k-32-mixed", "kind": "sample", "n": 32, "vocab": 128256, "temperature": 1.0, "top_k": 0,
         "top_p": 1.0, "min_p": 0.0, "mixed": True, "bulk": 2.0, "spread": 11},
        # a large batch of flat distributions, the nucleus of each
        {"name": "sample-128k-256-top-p", "kind": "sample", "n": 256, "vocab": 128256, "temperature": 0.9, "top_k": 0,
         "top_p": 0.9, "min_p": 0.0, "mixed": False, "bulk": 2.5, "spread": 12},
    ]


def _log(rng, low, high):
    """An integer from low to high, evenly over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["score", "score", "score", "score", "rotate", "rotate", "read", "sample", "sample"])
    spread = rng.randrange(1 << 30)
    if kind == "sample":
        vocab = rng.choice([32000, 128256, _log(rng, 1000, 128256)])
        n = _log(rng, 1, max(1, min(256, 256 * 128256 // vocab)))
        return {"kind": kind, "n": n, "vocab": vocab, "temperature": rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]),
                "top_k": rng.choice([0, 0, 1, _log(rng, 2, 100), _log(rng, 100, vocab)]),
                "top_p": rng.choice([1.0, 0.5, 0.9, 0.99]), "min_p": rng.choice([0.0, 0.0, 0.02, 0.2]),
                "mixed": rng.random() < 0.4, "bulk": rng.choice([0.5, 1.0, 2.0, 3.0]), "spread": spread}
    heads, kvh, dim = shape = rng.choice([SMOL, L1B, L1B, L8B, L8B, L70B, TINY])
    block = rng.choice([16, 16, 16, 32, 64])
    base = {"kind": kind, **_shape(shape), "block": block, "q8": rng.random() < 0.4, "spread": spread}
    if kind == "rotate":
        return {**base, "n": _log(rng, 1, 3000 * 6144 // ((heads + 2 * kvh) * dim)), "norm": rng.random() < 0.6,
                "interleaved": rng.random() < 0.5, "rotary": rng.choice([dim, dim, dim // 2]),
                "far": _log(rng, 100, 131072)}
    if kind == "read":
        layers = rng.randrange(1, 9)
        return {**base, "n": _log(rng, 1, 6000 * 1024 // (layers * kvh * dim)), "layers": layers}
    rows = rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 16, 1500)])
    n = _log(rng, 1, 64 if rows < 16 else 6)
    most = min(32768, int(4e10 / (4 * heads * dim * n * rows)), int(1.0e9 / (8 * kvh * dim * n)))
    mean = max(_log(rng, 1, max(2, most)), rows)
    low = max(rows, int(mean * rng.choice([1.0, 0.6, 0.2])))
    style = rng.choice(["", "window", "window", "prefix", "document"])
    return {**base, "n": n, "low": low, "high": max(low, 2 * mean - low), "rlow": max(1, int(rows * rng.uniform(0.2, 1))),
            "rhigh": rows, "cap": rng.choice([0.0, 0.0, 20.0, 50.0]), "slopes": rng.random() < 0.4,
            "window": _log(rng, 1, 2 * mean) if style == "window" else 0,
            "prefix": _log(rng, 1, 2 * mean) if style == "prefix" else 0,
            "document": _log(rng, 8, 2 * mean + 8) if style == "document" else 0}


# ------------------------------------------------------------------ sizes

def _ints(case, low, high, tag):
    r = random.Random(case["spread"] * 8 + tag)
    return [r.randint(case[low], case[high]) for _ in range(case["n"])]


def _lengths(case):
    return _ints(case, "low", "high", 0)


def _rows(case):
    return [min(r, n) for r, n in zip(_ints(case, "rlow", "rhigh", 1), _lengths(case))]


def _ranges(case):
    """Per sequence its rows' positions, and the first key and the end of the keys
    that each may see: the text up to itself, a prefix whole, a window back from
    itself or to its document's first token."""
    out = []
    for n, r in zip(_lengths(case), _rows(case)):
        pos = np.arange(n - r, n)
        first, end = np.zeros(r, np.int64), pos + 1
        if case["window"]:
            first = np.maximum(first, pos + 1 - case["window"])
        if case["document"]:
            first = np.maximum(first, pos // case["document"] * case["document"])
        if case["prefix"]:  # rows of the prefix see all of it
            end = np.where(pos < case["prefix"], min(n, case["prefix"]), end)
        out.append((pos, first, end))
    return out


def work(case):
    kind = case["kind"]
    if kind == "sample":
        elements = case["n"] * case["vocab"]
        return {"bytes": 4 * elements + 28 * case["n"], "flops": 4 * elements}
    element = 34 / 32 if case["q8"] else 4
    kvw, hidden = case["kv_heads"] * case["dim"], case["heads"] * case["dim"]
    if kind == "read":
        return {"bytes": case["n"] * (case["layers"] * 2 * kvw * (4 + element) + 8), "flops": case["n"] * case["layers"] * 2 * kvw}
    if kind == "rotate":
        back = 2 * kvw * (4 + element) if case["q8"] else 0
        return {"bytes": case["n"] * ((2 * hidden + 2 * kvw) * 4 + 2 * kvw * element + back + 12),
                "flops": 6 * case["n"] * (hidden + kvw)}
    keys = pairs = rows = 0
    for pos, first, end in _ranges(case):
        keys += int(end.max() - first.min())
        pairs += int((end - first).sum())
        rows += len(pos)
    return {"bytes": keys * 2 * kvw * element + rows * 2 * hidden * 4, "flops": 4 * hidden * pairs}


# ------------------------------------------------------------------- data

def _gen(seed, *tags):
    g = torch.Generator(device=DEVICE)
    g.manual_seed((int(seed) * 1000003 + zlib.crc32(repr(tags).encode())) % (1 << 62))
    return g


def _normal(seed, tag, *shape):
    return torch.randn(*shape, generator=_gen(seed, tag), device=DEVICE)


def _kv_rows(case, seed, which, rows, layers=1):
    """[rows, layers * kv_width]: normal, each channel of a key at a scale of its own."""
    w = layers * case["kv_heads"] * case["dim"]
    scale = torch.exp(0.4 * _normal(seed, "scale", w)) if which == "k" else 1.0
    return _normal(seed, which, rows, w) * scale


def _order(case, lengths):
    """(sequence, token) of every append: blocks of the sequences in turn, as
    sequences that grow side by side take them from the pool."""
    r = np.random.default_rng(case["spread"])
    seq, tok = [np.zeros(0, int)], [np.zeros(0, int)]
    b = case["block"]
    for lo in range(0, max(lengths), b):
        live = np.array([i for i, n in enumerate(lengths) if n > lo], dtype=np.int64)
        for i in r.permutation(live):
            t = np.arange(lo, min(lo + b, lengths[i]))
            seq.append(np.full(t.size, i))
            tok.append(t)
    return np.concatenate(seq), np.concatenate(tok)


def _tables(case, lengths):
    """[n, most blocks] ids, 0 behind a sequence's own: an empty pool hands out
    0, 1, ... in the order of the appends."""
    b = case["block"]
    table = np.zeros((len(lengths), max(1, -(-max(lengths) // b))), np.int64)
    seq, tok = _order(case, lengths)
    fresh = tok % b == 0
    table[seq[fresh], tok[fresh] // b] = np.arange(int(fresh.sum()))
    return table


def _blocks(case, lengths):
    return sum(-(-n // case["block"]) for n in lengths)


def _encode(x):
    """Q8_0 of [..., 32k] f32 values: (int8 of x's shape, fp16 scale of each 32)."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    scale = g.abs().amax(-1, keepdim=True).double() / 127
    q = (g.double() / scale.float().double()).float()
    q = torch.where(scale == 0, torch.zeros_like(q), torch.round(q).clamp(-127, 127))
    return q.to(torch.int8).reshape(x.shape), scale.half()[..., 0]


def _decode(q, scale):
    g = q.float().reshape(*q.shape[:-1], -1, 32) * scale.float()[..., None]
    return g.reshape(q.shape)


def _held(x, q8):
    """What the cache holds of f32 rows, as float64."""
    if not q8:
        return x.double()
    g = x.reshape(x.shape[0], -1, 32)
    top = g.abs().amax(2, keepdim=True).double() / 127
    ints = torch.where(top > 0, (g.double() / top.float().double().clamp(min=1e-300)).float(), torch.zeros_like(g))
    return (torch.round(ints).clamp(-127, 127).double() * top.half().double()).reshape(x.shape)


def _pool(case, blocks, layers):
    """Empty blocks in plain tensors, [blocks, layers, 2, block, kv_width]: f32, or int8 and fp16 scales."""
    shape = (blocks, layers, 2, case["block"], case["kv_heads"] * case["dim"])
    if not case["q8"]:
        return torch.zeros(shape, device=DEVICE)
    return (torch.zeros(shape, dtype=torch.int8, device=DEVICE),
            torch.zeros(*shape[:-1], shape[-1] // 32, dtype=torch.float16, device=DEVICE))


def _put(pool, case, slots, rows):
    """rows [n, layers, 2, kv_width] into slots."""
    blk, slot = slots // case["block"], slots % case["block"]
    if not case["q8"]:
        pool[blk, :, :, slot] = rows
        return
    q, s = _encode(rows)
    pool[0][blk, :, :, slot] = q
    pool[1][blk, :, :, slot] = s


def _get(pool, case, slots):
    """[n, layers, 2, kv_width] f32 out of slots."""
    blk, slot = slots // case["block"], slots % case["block"]
    if not case["q8"]:
        return pool[blk, :, :, slot]
    return _decode(pool[0][blk, :, :, slot], pool[1][blk, :, :, slot])


def _cache(st, case, lengths, layers, k, v):
    """The framework's cache with rows k and v of the sequences in the same blocks."""
    from tvara_amd import kv

    st.cache = kv.PagedCache(layers, case["kv_heads"], case["dim"], case["block"], _blocks(case, lengths),
                             kv.Q8_0 if case["q8"] else kv.F32)
    st.seqs = np.array([st.cache.create_sequence() for _ in lengths], dtype=np.uint64)
    seq, tok = _order(case, lengths)
    first = np.concatenate([[0], np.cumsum(lengths)[:-1]])
    rows = torch.from_numpy(first[seq] + tok).to(DEVICE)
    k, v = k[rows], v[rows]
    torch.cuda.synchronize()
    ids = st.seqs[seq]
    for lo in range(0, ids.size, 1 << 16):
        part = np.ascontiguousarray(ids[lo:lo + (1 << 16)])
        st.cache.append_batch_device(part, k[lo:].data_ptr(), v[lo:].data_ptr())
    st.cache.synchronize()


def _pool_of(cache, case, layers):
    """The cache's own f32 blocks as a torch tensor, laid out as in _pool."""
    base, stride = cache.pool_address()

    class Memory:  # the tensor holds it, and so the cache, for as long as the blocks are looked at
        __cuda_array_interface__ = {"shape": (cache.max_blocks * stride,), "typestr": "|u1", "data": (base, False),
                                    "version": 2}

    memory = Memory()
    memory.owner = cache
    raw = torch.as_tensor(memory, device=DEVICE)
    b, w = case["block"], case["kv_heads"] * case["dim"]
    return raw.view(torch.float32).as_strided((cache.max_blocks, layers, 2, b, w), (stride // 4, 2 * b * w, b * w, w, 1))


class _State:
    pass


# ------------------------------------------------------------------ score

def _slopes(case):
    """A distance's weight for each head, falling by powers of two over the heads."""
    h = case["heads"]
    return np.array([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], np.float32)


def _prepare_score(st, case, seed):
    lengths, rows, ranges = _lengths(case), _rows(case), _ranges(case)
    k, v = (_kv_rows(case, seed, which, sum(lengths)) for which in ("k", "v"))
    st.q = 1.5 * _normal(seed, "q", sum(rows), case["heads"] * case["dim"])
    st.slopes = _slopes(case) if case["slopes"] else None
    pos, first, end = (np.concatenate(x) for x in zip(*ranges))
    if own:
        from tvara_amd import attention

        _cache(st, case, lengths, 1, k, v)
        st.out = torch.empty_like(st.q)
        starts = [n - r for n, r in zip(lengths, rows)]
        st.plan = attention.ScorePlan(st.cache, st.seqs, starts, rows, case["heads"], CONTEXT, first=first, end=end,
                                      cap=case["cap"], slopes=st.slopes)
        return st
    table = _tables(case, lengths)
    st.pool = _pool(case, _blocks(case, lengths), 1)
    at = np.repeat(np.arange(case["n"]), lengths)
    tok = np.concatenate([np.arange(n) for n in lengths])
    slots = table[at, tok // case["block"]] * case["block"] + tok % case["block"]
    kvw = k.shape[1]
    _put(st.pool, case, torch.from_numpy(slots).to(DEVICE), torch.stack([k, v], 1).reshape(-1, 1, 2, kvw))
    st.table = torch.from_numpy(table).to(DEVICE)
    st.longest, st.most = max(lengths), max(rows)
    row0 = np.concatenate([[0], np.cumsum(rows)[:-1]])
    pad = np.minimum(row0[:, None] + np.arange(st.most), sum(rows) - 1)
    flat = np.concatenate([i * st.most + np.arange(r) for i, r in enumerate(rows)])
    st.pad, st.flat, st.pos, st.first, st.end = (torch.from_numpy(np.ascontiguousarray(x)).to(DEVICE)
                                                 for x in (pad, flat, pos, first, end))
    return st


def _plain_score(st):
    case = st.case
    heads, kvh, d, n, most = case["heads"], case["kv_heads"], case["dim"], case["n"], st.most
    g = heads // kvh
    q = st.q.reshape(-1, kvh, g, d)[st.pad].permute(0, 2, 3, 1, 4).reshape(n, kvh, g * most, d)
    key = torch.arange(st.longest, device=q.device)
    slots = st.table[:, key // case["block"]] * case["block"] + key % case["block"]
    kv = _get(st.pool, case, slots)[:, :, 0].reshape(n, st.longest, 2, kvh, d)
    s = torch.matmul(q, kv[:, :, 0].permute(0, 2, 3, 1).contiguous()) / math.sqrt(d)
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    s = s.reshape(n, kvh, g, most, st.longest)
    if case["slopes"]:
        away = (st.pos[st.pad][:, :, None] - key).abs().float()
        slope = torch.from_numpy(st.slopes).to(q.device).reshape(kvh, g, 1, 1)
        s = s - slope * away[:, None, None]
    seen = (key >= st.first[st.pad][:, :, None]) & (key < st.end[st.pad][:, :, None])
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-37)
    o = torch.matmul(p.reshape(n, kvh, g * most, st.longest), kv[:, :, 1].permute(0, 2, 1, 3).contiguous())
    return o.reshape(n, kvh, g, most, d).permute(0, 3, 1, 2, 4).reshape(n * most, heads * d)[st.flat]


def _exact_score(case, seed):
    lengths, rows, ranges = _lengths(case), _rows(case), _ranges(case)
    heads, kvh, d = case["heads"], case["kv_heads"], case["dim"]
    k, v = (_kv_rows(case, seed, which, sum(lengths)) for which in ("k", "v"))
    q = 1.5 * _normal(seed, "q", sum(rows), heads * d)
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEVICE)
    slopes, g = _slopes(case), heads // kvh
    c0 = r0 = 0
    for n, r, (pos, first, end) in zip(lengths, rows, ranges):
        kk, vv = (_held(x[c0:c0 + n], case["q8"]).reshape(n, kvh, d) for x in (k, v))
        at = np.arange(n)
        hidden = torch.from_numpy((at < first[:, None]) | (at >= end[:, None])).to(DEVICE)
        away = torch.from_numpy(np.abs(pos[:, None] - at)).to(DEVICE).double()
        for h in range(heads):
            s = torch.mm(q[r0:r0 + r, h * d:(h + 1) * d].double(), kk[:, h // g].t().contiguous()) / math.sqrt(d)
            if case["cap"]:
                s = torch.tanh(s / case["cap"]) * case["cap"]
            if case["slopes"]:
                s -= float(slopes[h]) * away
            s[hidden] = -math.inf
            out[r0:r0 + r, h * d:(h + 1) * d] = torch.mm(torch.softmax(s, 1), vv[:, h // g].contiguous())
        c0, r0 = c0 + n, r0 + r
    return out


# ----------------------------------------------------------------- rotate

def _rotary_inputs(case, seed):
    """Rows of a fused product (queries, keys, values side by side), positions, frequencies, weights."""
    n, d = case["n"], case["dim"]
    kvw, hidden = case["kv_heads"] * d, case["heads"] * d
    qkv = _normal(seed, "qkv", n, hidden + 2 * kvw)
    pos = torch.randint(0, case["far"], (n,), generator=_gen(seed, "positions"), device=DEVICE, dtype=torch.int32)
    half = case["rotary"] // 2
    freqs = torch.from_numpy((10000.0 ** (-np.arange(half) / half)).astype(np.float32)).to(DEVICE)
    wq, wk = (1 + 0.2 * _normal(seed, which, d) for which in ("wq", "wk"))
    return qkv, pos, freqs, wq, wk


def _slots_of(case):
    """A slot for each row, blocks in no order; a padded batch's last rows have none."""
    n, b = case["n"], case["block"]
    order = np.random.default_rng(case["spread"]).permutation(-(-n // b))
    at = np.arange(n)
    slots = order[at // b] * b + at % b
    if n >= 16:
        slots[-(n // 16):] = -1
    return slots


def _empty_cache(st, case, layers):
    from tvara_amd import kv

    st.cache = kv.PagedCache(layers, case["kv_heads"], case["dim"], case["block"], -(-case["n"] // case["block"]),
                             kv.Q8_0 if case["q8"] else kv.F32)
    st.seqs = np.array([st.cache.create_sequence()], dtype=np.uint64)
    st.cache.reserve(st.seqs, [st.cache.max_blocks * case["block"]])
    st.plan = kv.SlotPlan(st.cache, st.seqs)


def _prepare_rotate(st, case, seed):
    st.qkv, st.pos, st.freqs, st.wq, st.wk = _rotary_inputs(case, seed)
    kvw, hidden = case["kv_heads"] * case["dim"], case["heads"] * case["dim"]
    slots = _slots_of(case)
    st.slots = torch.from_numpy(slots).to(DEVICE)
    st.q = torch.empty(case["n"], hidden, device=DEVICE)
    st.keys, st.values = (torch.zeros(case["n"], kvw, device=DEVICE) for _ in "kv")
    if own:
        _empty_cache(st, case, 1)
        st.pool = None if case["q8"] else _pool_of(st.cache, case, 1)
    else:
        st.pool = _pool(case, -(-case["n"] // case["block"]), 1)
        st.live = torch.from_numpy(np.flatnonzero(slots >= 0)).to(DEVICE)
    return st


def _turn(x, case, weight, cos, sin, eps=1e-6):
    """[n, heads, dim] normalised head by head and rotated, in float64."""
    x, r = x.double(), case["rotary"]
    if case["norm"]:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y, x[..., r:]], -1)


def _plain_rotate(st):
    case, n = st.case, st.case["n"]
    hidden, kvw, d = st.q.shape[1], st.keys.shape[1], case["dim"]
    angle = st.pos.double()[:, None] * st.freqs.double()
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    q = _turn(st.qkv[:, :hidden].reshape(n, -1, d), case, st.wq, cos, sin).float().reshape(n, hidden)
    k = _turn(st.qkv[:, hidden:hidden + kvw].reshape(n, -1, d), case, st.wk, cos, sin).float().reshape(n, kvw)
    rows = torch.stack([k, st.qkv[:, hidden + kvw:]], 1)[st.live][:, None]
    slots = st.slots[st.live]
    _put(st.pool, case, slots, rows)
    if not case["q8"]:
        return q, st.pool
    back = _get(st.pool, case, slots)
    st.keys[st.live], st.values[st.live] = back[:, 0, 0], back[:, 0, 1]
    return q, st.keys, st.values


def _own_rotate(st):
    case, n = st.case, st.case["n"]
    hidden, kvw = st.q.shape[1], st.keys.shape[1]
    at, width = st.qkv.data_ptr(), st.qkv.shape[1]
    norm = {"q_norm_ptr": st.wq.data_ptr(), "k_norm_ptr": st.wk.data_ptr(), "eps": 1e-6} if case["norm"] else {}
    st.plan.rotate(st.slots.data_ptr(), n, 0, at, at + 4 * hidden, at + 4 * (hidden + kvw), st.pos.data_ptr(),
                   st.freqs.data_ptr(), case["rotary"], case["heads"], st.q.data_ptr(), q_stride=width, kv_stride=width,
                   interleaved=case["interleaved"], **norm)
    if not case["q8"]:
        return st.q, st.pool
    st.plan.read(st.slots.data_ptr(), n, 0, 1, st.keys.data_ptr(), st.values.data_ptr(), kvw, 0)
    return st.q, st.keys, st.values


def _exact_rotate(case, seed):
    qkv, pos, freqs, wq, wk = _rotary_inputs(case, seed)
    d, r, slots = case["dim"], case["rotary"], _slots_of(case)
    kvw, hidden = case["kv_heads"] * d, case["heads"] * d
    x = qkv.double().reshape(case["n"], -1, d)
    heads = x[:, :case["heads"] + case["kv_heads"]]
    if case["norm"]:
        rms = (heads.square().sum(-1, keepdim=True) / d + 1e-6).sqrt()
        heads = heads / rms
        heads = torch.cat([heads[:, :case["heads"]] * wq.double(), heads[:, case["heads"]:] * wk.double()], 1)
    # pair j turns as a complex number
    lo = np.arange(0, r, 2) if case["interleaved"] else np.arange(r // 2)
    hi = lo + (1 if case["interleaved"] else r // 2)
    z = torch.complex(heads[..., lo], heads[..., hi]) * torch.polar(torch.ones_like(freqs).double(), freqs.double() * pos.double()[:, None])[:, None]
    heads = heads.clone()
    heads[..., lo], heads[..., hi] = z.real, z.imag
    q, k = heads[:, :case["heads"]].reshape(-1, hidden), heads[:, case["heads"]:].reshape(-1, kvw)
    v = x[:, case["heads"] + case["kv_heads"]:].reshape(-1, kvw)
    live = np.flatnonzero(slots >= 0)
    if case["q8"]:
        out = []
        for rows in (k, v):
            back = torch.zeros_like(rows)
            back[live] = _held(rows[live].float(), True)
            out.append(back)
        return q, *out
    blocks, b = -(-case["n"] // case["block"]), case["block"]
    pool = torch.zeros(blocks * b, 2, kvw, dtype=torch.float64, device=DEVICE)
    pool[slots[live], 0], pool[slots[live], 1] = k[live], v[live]
    return q, pool.reshape(blocks, b, 2, kvw).transpose(1, 2).reshape(blocks, 1, 2, b, kvw)


# ------------------------------------------------------------------- read

def _prepare_read(st, case, seed):
    n, layers = case["n"], case["layers"]
    kvw = case["kv_heads"] * case["dim"]
    k, v = (_kv_rows(case, seed, which, n, layers).reshape(n, layers, kvw) for which in ("k", "v"))
    st.slots = torch.from_numpy(_slots_of(case)).to(DEVICE)
    # (a read of slots that were written: the batch's padding has no slot)
    st.live = torch.nonzero(st.slots >= 0)[:, 0]
    st.keys, st.values = (torch.zeros(n, layers, kvw, device=DEVICE) for _ in "kv")
    if own:
        _empty_cache(st, case, layers)
        torch.cuda.synchronize()
        st.plan.write(st.slots.data_ptr(), None, n, k.data_ptr(), v.data_ptr(), n, layers * kvw, kvw)
        st.cache.synchronize()
    else:
        st.pool = _pool(case, -(-n // case["block"]), layers)
        _put(st.pool, case, st.slots[st.live], torch.stack([k, v], 2)[st.live])
    return st


def _plain_read(st):
    rows = _get(st.pool, st.case, st.slots[st.live])
    st.keys[st.live], st.values[st.live] = rows[:, :, 0], rows[:, :, 1]
    return st.keys, st.values


def _own_read(st):
    n, layers, kvw = st.keys.shape
    st.plan.read(st.slots.data_ptr(), n, 0, layers, st.keys.data_ptr(), st.values.data_ptr(), layers * kvw, kvw)
    return st.keys, st.values


def _exact_read(case, seed):
    n, layers = case["n"], case["layers"]
    live = np.flatnonzero(_slots_of(case) >= 0)
    out = []
    for which in ("k", "v"):
        rows = _kv_rows(case, seed, which, n, layers)
        back = torch.zeros_like(rows, dtype=torch.float64)
        back[live] = _held(rows[live], case["q8"])
        out.append(back.reshape(n, layers, -1))
    return tuple(out)


# ----------------------------------------------------------------- sample

def _asked(case):
    """Each row's temperature, top-k (0: all), top-p and min-p."""
    n = case["n"]
    t, k, p, m = (np.full(n, case[x]) for x in ("temperature", "top_k", "top_p", "min_p"))
    if case["mixed"]:
        r = random.Random(case["spread"])
        for i in range(n):
            t[i] = r.choice([0.0, 0.6, 0.8, 1.0, 1.2])
            k[i] = r.choice([0, 0, 20, 50, 200])
            p[i] = r.choice([1.0, 1.0, 0.8, 0.95])
            m[i] = r.choice([0.0, 0.0, 0.05])
    return t.astype(np.float32), k.astype(np.int32), p.astype(np.float32), m.astype(np.float32)


def _texts(case, seed):
    """Logits as a bf16 model gives them (ties among them): a bulk, and a few tokens
    above it by more or less; and a random number in [0, 1) for each row."""
    n, v = case["n"], case["vocab"]
    x = case["bulk"] * _normal(seed, "logits", n, v)
    likely = torch.randint(0, v, (n, 24), generator=_gen(seed, "likely"), device=DEVICE)
    lift = torch.rand(n, 24, generator=_gen(seed, "lift"), device=DEVICE)
    sure = torch.rand(n, 1, generator=_gen(seed, "sure"), device=DEVICE)
    x.scatter_add_(1, likely, 16 * sure * lift)
    u = torch.rand(n, generator=_gen(seed, "u"), device=DEVICE)
    return x.bfloat16().float(), u


def _prepare_sample(st, case, seed):
    st.logits, st.u = _texts(case, seed)
    st.t, st.k, st.p, st.m = (torch.from_numpy(x).to(DEVICE) for x in _asked(case))
    if own:
        from tvara_amd import sampling

        st.tokens = torch.empty(case["n"], dtype=torch.int32, device=DEVICE)
        st.chances = torch.empty(case["n"], device=DEVICE)
        st.plan = sampling.SamplePlan(case["n"], case["vocab"])
    return st


def _plain_sample(st):
    """By sorting: values down, the lowest index first among equals."""
    x, order = torch.sort(st.logits, dim=1, descending=True, stable=True)
    v = x.shape[1]
    cold = st.t == 0
    t = torch.where(cold, 1.0, st.t).double()[:, None]
    k = torch.where(cold, 1, torch.where(st.k == 0, v, st.k))[:, None]
    w = torch.exp((x.double() - x[:, :1].double()) / t)
    w = torch.where(torch.arange(v, device=x.device) < k, w, 0.0)
    upto = torch.cumsum(w, 1)
    keep = (upto - w < st.p.double()[:, None] * upto[:, -1:]) & (w >= st.m.double()[:, None])
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    upto = torch.cumsum(w, 1)
    token = torch.searchsorted(upto, (st.u.double() * upto[:, -1])[:, None], right=True).clamp(max=v - 1)
    return token[:, 0].int(), (torch.gather(w, 1, token) / upto[:, -1:])[:, 0].float()


def _own_sample(st):
    st.plan.launch(st.logits.data_ptr(), st.u.data_ptr(), st.tokens.data_ptr(), st.chances.data_ptr(),
                   temperature_ptr=st.t.data_ptr(), top_k_ptr=st.k.data_ptr(), top_p_ptr=st.p.data_ptr(),
                   min_p_ptr=st.m.data_ptr())
    return st.tokens, st.chances


def _exact_sample(case, seed):
    logits, us = _texts(case, seed)
    out = torch.zeros(case["n"], dtype=torch.float64, device=DEVICE)
    for i, (t, k, p, m) in enumerate(zip(*_asked(case))):
        x = logits[i].double()
        if t == 0:
            out[i] = 1.0
            continue
        order = torch.argsort(x, descending=True, stable=True)[:int(k) if k else None]
        w = torch.softmax((x[order] - x.max()) / float(t), 0)
        enough = (torch.cumsum(w, 0) - w) < float(p)
        order, w = order[enough], w[enough]
        likely = w >= float(m) * w[0]
        order, w = order[likely], w[likely] / w[likely].sum()
        by_index = torch.argsort(order)
        at = (torch.cumsum(w[by_index], 0) <= float(us[i])).sum().clamp(max=w.numel() - 1)
        out[i] = w[by_index][at]
    return out


# -------------------------------------------------------------- the calls

def prepare(case, seed):
    st = _State()
    st.case = case
    return {"score": _prepare_score, "rotate": _prepare_rotate, "read": _prepare_read,
            "sample": _prepare_sample}[case["kind"]](st, case, seed)


def _own_score(st):
    st.plan.launch(0, st.q.data_ptr(), st.out.data_ptr())
    return st.out


def run(st):
    calls = ({"score": _own_score, "rotate": _own_rotate, "read": _own_read, "sample": _own_sample} if own else
             {"score": _plain_score, "rotate": _plain_rotate, "read": _plain_read, "sample": _plain_sample})
    return calls[st.case["kind"]](st)


def exact(case, seed):
    """run()'s answer in 64 bits; whole numbers have none."""
    if case["kind"] == "sample":
        return None, _exact_sample(case, seed)
    return {"score": _exact_score, "rotate": _exact_rotate, "read": _exact_read}[case["kind"]](case, seed)
