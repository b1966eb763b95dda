"""What speculative decoding with trees of drafted tokens is timed on: attention
of the trees over the paged KV cache, the greedy acceptance of their tokens,
the slot maps and block tables of the rows to come, and the write of the
accepted rows, each alone and in a step together.

``listed()`` names the cases and ``draw()`` gives others of the same ranges.  A
case is a plain dict; sequence lengths, tree shapes and block orders follow from
its own fields, every value that is computed on from the seed.  Five kinds:

tree     one ``TreePlan.launch``: every drafted node of every sequence attends
         to the sequence's cached tokens, its ancestors and itself, one layer.
accept   one ``TreePlan.accept``: which nodes the model's own greedy choices
         confirm, and the token that follows them.
slots    one ``SlotPlan.build``: offsets, positions, slots and padded block
         tables of a batch from its lengths.
write    one ``SlotPlan.write``: rows of K and V, all layers, into slots.
step     all of it for one step of a batch: room taken, plans, every layer's
         attention, acceptance, slot map and write; rolled back at the end.

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
        # one user's stream on a small model, a small tree: launch-bound
        {"name": "tree-smol-1x512x8", "kind": "tree", **_shape(SMOL), "n": 1, "low": 512, "high": 512, "tlow": 8,
         "thigh": 8, "width": 4, "block": 16, "q8": False, "precision": "f32", "spread": 1},
        # a serving batch of unequal contexts and trees, the default precision
        {"name": "tree-1b-f32-ragged", "kind": "tree", **_shape(L1B), "n": 16, "low": 100, "high": 3000, "tlow": 3,
         "thigh": 24, "width": 5, "block": 16, "q8": False, "precision": "f32", "spread": 2},
        # a larger model's batch with trees of 32
        {"name": "tree-8b-x3-16x4096x32", "kind": "tree", **_shape(L8B), "n": 16, "low": 4096, "high": 4096,
         "tlow": 32, "thigh": 32, "width": 8, "block": 16, "q8": False, "precision": "f32x3", "spread": 3},
        # few long contexts over quantised blocks of 64 tokens
        {"name": "tree-8b-q8-x3-long", "kind": "tree", **_shape(L8B), "n": 4, "low": 20000, "high": 32768, "tlow": 13,
         "thigh": 29, "width": 6, "block": 64, "q8": True, "precision": "f32x3", "spread": 4},
        # wide groups and large trees: the most arithmetic
        {"name": "tree-70b-x3-8x4096x64", "kind": "tree", **_shape(L70B), "n": 8, "low": 4000, "high": 4200, "tlow": 64,
         "thigh": 64, "width": 16, "block": 16, "q8": False, "precision": "f32x3", "spread": 5},
        # one user's small tree
        {"name": "accept-32k-1x8", "kind": "accept", "n": 1, "tlow": 8, "thigh": 8, "width": 3, "vocab": 32000,
         "agree": 0.7, "spread": 6},
        # a batch's trees over a large vocabulary
        {"name": "accept-128k-32x16", "kind": "accept", "n": 32, "tlow": 12, "thigh": 20, "width": 4, "vocab": 128256,
         "agree": 0.7, "spread": 7},
        # one request's next tokens
        {"name": "slots-1x5", "kind": "slots", "n": 1, "low": 513, "high": 513, "clow": 5, "chigh": 5, "block": 16,
         "stride": 0, "spread": 8},
        # a large batch of prompts and continuations, packed
        {"name": "slots-256-packed", "kind": "slots", "n": 256, "low": 0, "high": 4096, "clow": 0, "chigh": 700,
         "block": 16, "stride": 0, "spread": 9},
        # a batch's accepted tokens over 16 layers, f32 blocks, one row a node for all layers
        {"name": "write-1b-64x16-layers", "kind": "write", **_shape(L1B), "n": 64, "low": 50, "high": 200, "clow": 1,
         "chigh": 6, "layers": 16, "by_layer": False, "block": 16, "q8": False, "spread": 10},
        # the same over quantised blocks, the model's layer-by-layer rows
        {"name": "write-8b-q8-32x8-layers", "kind": "write", **_shape(L8B), "n": 32, "low": 50, "high": 200, "clow": 0,
         "chigh": 7, "layers": 8, "by_layer": True, "block": 32, "q8": True, "spread": 11},
        # one whole step of a batch over four layers
        {"name": "step-1b-16x4-layers", "kind": "step", **_shape(L1B), "n": 16, "low": 200, "high": 2000, "tlow": 6,
         "thigh": 16, "width": 4, "layers": 4, "block": 16, "q8": False, "precision": "f32x3", "vocab": 32000,
         "agree": 0.7, "spread": 12},
    ]


def _log(rng, low, high):
    """An integer from low to high, evenly over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "tree", "accept", "slots", "write", "step"])
    spread = rng.randrange(1 << 30)
    if kind == "accept":
        vocab = rng.choice([32000, 128256, _log(rng, 1000, 128256)])
        t = _log(rng, 1, 64)
        n = _log(rng, 1, max(1, min(64, 512 * 128256 // (t * vocab))))
        return {"kind": kind, "n": n, "tlow": max(1, t // 2), "thigh": t, "width": rng.randrange(1, 9), "vocab": vocab,
                "agree": rng.choice([0.3, 0.7, 0.95]), "spread": spread}
    block = rng.choice([16, 16, 16, 32, 64])
    if kind == "slots":
        n = _log(rng, 1, 256)
        low, count = rng.choice([0, _log(rng, 1, 2000)]), _log(rng, 1, 700)
        stride = rng.choice([0, 0, count])
        return {"kind": kind, "n": n, "low": low, "high": low + _log(rng, 1, 2000), "clow": rng.randrange(0, count + 1),
                "chigh": count, "block": block, "stride": stride, "spread": spread}
    if kind == "write":
        shape = rng.choice([SMOL, L1B, L8B, TINY])
        low, count = _log(rng, 1, 200), _log(rng, 1, 8)
        return {"kind": kind, **_shape(shape), "n": _log(rng, 1, 64), "low": low, "high": low + _log(rng, 1, 100),
                "clow": rng.randrange(0, count + 1), "chigh": count, "layers": rng.randrange(1, 9),
                "by_layer": rng.random() < 0.5, "block": block, "q8": rng.random() < 0.4, "spread": spread}
    q8 = rng.random() < 0.4
    t = _log(rng, 1, 64)
    precision = rng.choice(["f32", "f32x3"])
    if kind == "step":
        low = _log(rng, 1, 1000)
        return {"kind": kind, **_shape(rng.choice([SMOL, L1B, TINY])), "n": _log(rng, 1, 24), "low": low,
                "high": low + _log(rng, 1, 1000), "tlow": max(1, t // 4), "thigh": max(1, t // 2),
                "width": rng.randrange(1, 9), "layers": rng.randrange(1, 5), "block": block, "q8": q8,
                "precision": precision, "vocab": 32000, "agree": 0.7, "spread": spread}
    heads, kvh, dim = rng.choice([SMOL, L1B, L1B, L8B, L8B, L70B, TINY])
    n = _log(rng, 1, 64)
    most = 20e9 if precision == "f32" else 60e9  # flops of the largest drawn tree batch
    mean = min(32768, int(most / (4 * heads * dim * n * t)), int(1.0e9 / (8 * kvh * dim * n)))
    mean = _log(rng, 1, max(2, mean))
    low = max(0, int(mean * rng.choice([1.0, 0.5, 0.0])))
    return {"kind": kind, "heads": heads, "kv_heads": kvh, "dim": dim, "n": n, "low": low, "high": 2 * mean - low,
            "tlow": max(1, int(t * rng.uniform(0.3, 1))), "thigh": t, "width": rng.randrange(1, 17), "block": block,
            "q8": q8, "precision": precision, "spread": spread}


# ------------------------------------------------------------------ sizes

def _ints(case, low, high, tag):
    r = random.Random(case["spread"] * 8 + tag)
    return [r.randint(case[low], case[high]) for _ in range(case["n"])]


def _lengths(case):
    return _ints(case, "low", "high", 0)


def _counts(case):
    return _ints(case, "clow", "chigh", 1)


def _trees(case):
    """The parents of every tree's nodes: within the `width` nodes before, the
    first a root, now and then another."""
    r = random.Random(case["spread"] * 8 + 3)
    out = []
    for t in _ints(case, "tlow", "thigh", 2):
        out.append([-1 if j == 0 or r.random() < 0.03 else r.randint(max(0, j - case["width"]), j - 1)
                    for j in range(t)])
    return out


def _depths(parents):
    d = []
    for p in parents:
        d.append(1 if p < 0 else d[p] + 1)
    return d


def work(case):
    kind = case["kind"]
    if kind == "accept":
        rows = sum(len(t) for t in _trees(case))
        return {"bytes": rows * (case["vocab"] * 4 + 12), "flops": rows * case["vocab"]}
    if kind == "slots":
        total, blocks = sum(_counts(case)), _blocks(case)
        width = max(blocks)
        cap = case["n"] * case["stride"] if case["stride"] else total
        return {"bytes": 4 * sum(blocks) + 4 * case["n"] * width + 12 * cap + 12 * case["n"], "flops": total}
    element = 34 / 32 if case.get("q8") else 4
    kvw = case["kv_heads"] * case["dim"]
    if kind == "write":
        total = sum(_counts(case))
        return {"bytes": total * (case["layers"] * 2 * kvw * (4 + element) + 12), "flops": total * case["layers"] * 2 * kvw}
    hidden, trees, ctx = case["heads"] * case["dim"], _trees(case), _lengths(case)
    nodes = sum(len(t) for t in trees)
    pairs = sum(len(t) * c + sum(_depths(t)) for t, c in zip(trees, ctx))
    layers = case.get("layers", 1)
    b = layers * (sum(ctx) * 2 * kvw * element + nodes * (2 * kvw + 2 * hidden) * 4)
    f = layers * 4 * hidden * pairs
    if kind == "step":
        b += nodes * case["vocab"] * 4
        f += nodes * case["vocab"]
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------- data

def _gen(seed, *tags):
    g = torch.Generator(device=DEVICE)
    g.manual_seed((int(seed) * 1000003 + zlib.crc32(repr(tags).encode())) % (1 << 62))
    return g


def _kv_rows(case, seed, which, rows, layers=1):
    """[rows, layers * kv_width]: normal, each channel of a key at a scale of its own."""
    w = layers * case["kv_heads"] * case["dim"]
    scale = torch.exp(0.4 * torch.randn(w, generator=_gen(seed, "scale"), device=DEVICE)) if which.endswith("k") else 1.0
    return torch.randn(rows, w, generator=_gen(seed, which), device=DEVICE) * scale


def _blocks(case):
    """Blocks of each sequence: its tokens and, where more are to come, those."""
    more = _counts(case) if "clow" in case else [0] * case["n"]
    return [-(-(n + c) // case["block"]) for n, c in zip(_lengths(case), more)]


def _append_order(case, lengths):
    """(sequence, token) of every append: blocks of the sequences in turn, as
    sequences that grow side by side take them from the pool."""
    r = np.random.default_rng(case["spread"])
    seq, tok = [np.zeros(0, int)], [np.zeros(0, int)]
    b = case["block"]
    for lo in range(0, max(lengths, default=0), b):
        live = np.array([i for i, n in enumerate(lengths) if n > lo], dtype=np.int64)
        for i in r.permutation(live):
            t = np.arange(lo, min(lo + b, lengths[i]))
            seq.append(np.full(t.size, i))
            tok.append(t)
    return np.concatenate(seq), np.concatenate(tok)


def _tables(case):
    """[n, most blocks] ids, -1 behind a sequence's own: an empty pool hands
    out 0, 1, ... in the order of the appends, then the room for more tokens."""
    lengths, blocks, b = _lengths(case), _blocks(case), case["block"]
    table = np.full((case["n"], max(1, max(blocks))), -1, np.int64)
    seq, tok = _append_order(case, lengths)
    fresh = tok % b == 0
    table[seq[fresh], tok[fresh] // b] = np.arange(int(fresh.sum()))
    at = int(fresh.sum())
    for i, n in enumerate(lengths):
        have = -(-n // b)
        table[i, have:blocks[i]] = np.arange(at, at + blocks[i] - have)
        at += blocks[i] - have
    return table


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


class _State:
    pass


def _rows_of(case, table, layers):
    """Where the cached tokens lie in the pool: (block, slot), and their rows."""
    lengths = _lengths(case)
    first = np.concatenate([[0], np.cumsum(lengths)[:-1]]).astype(np.int64)
    seq = np.repeat(np.arange(case["n"]), lengths)
    pos = np.arange(sum(lengths)) - first[seq]
    blk = table[seq, pos // case["block"]]
    return torch.from_numpy(blk).to(DEVICE), torch.from_numpy(pos % case["block"]).to(DEVICE)


def _pool(case, k, v, table, layers):
    """The blocks in plain tensors: f32 [blocks, layers, 2, block, kv_width], or
    (int8 [blocks, layers, 2, kv heads, block, head_dim], fp16 scales [..., head_dim / 32])."""
    blocks, b = max(1, sum(_blocks(case))), case["block"]
    kvh, d = case["kv_heads"], case["dim"]
    blk, slot = _rows_of(case, table, layers)
    kv = torch.stack([k.reshape(-1, layers, kvh * d), v.reshape(-1, layers, kvh * d)], 2)
    if not case["q8"]:
        pool = torch.zeros(blocks, layers, 2, b, kvh * d, device=DEVICE)
        pool[blk, :, :, slot] = kv
        return pool
    q, s = _encode(kv)
    ints = torch.zeros(blocks, layers, 2, kvh, b, d, dtype=torch.int8, device=DEVICE)
    scales = torch.zeros(blocks, layers, 2, kvh, b, d // 32, dtype=torch.float16, device=DEVICE)
    ints[blk, :, :, :, slot] = q.reshape(-1, layers, 2, kvh, d)
    scales[blk, :, :, :, slot] = s.reshape(-1, layers, 2, kvh, d // 32)
    return ints, scales


def _cache(st, case, k, v, layers, spare=0):
    """The framework's cache with the same tokens in the same blocks."""
    from tvara_amd import kv

    lengths = _lengths(case)
    st.cache = kv.PagedCache(layers, case["kv_heads"], case["dim"], case["block"], max(1, sum(_blocks(case)) + spare),
                             kv.Q8_0 if case["q8"] else kv.F32)
    st.seqs = np.array([st.cache.create_sequence() for _ in lengths], dtype=np.uint64)
    st.lengths = np.array(lengths, dtype=np.uintp)
    seq, tok = _append_order(case, lengths)
    if seq.size:
        first = np.concatenate([[0], np.cumsum(lengths)[:-1]])
        rows = torch.from_numpy(first[seq] + tok).to(DEVICE)
        k, v = k[rows], v[rows]
        ids = st.seqs[seq]
        for lo in range(0, ids.size, 1 << 16):
            part = np.ascontiguousarray(ids[lo:lo + (1 << 16)])
            st.cache.append_batch_device(part, k[lo:].data_ptr(), v[lo:].data_ptr())
        st.cache.synchronize()


def _pool_of(cache, case, layers):
    """The cache's own blocks as torch tensors, laid out as in _pool."""
    base, stride = cache.pool_address()
    blocks = cache.max_blocks

    class Memory:  # the tensor holds it, and so the cache, for as long as the blocks are looked at
        __cuda_array_interface__ = {"shape": (blocks * stride,), "typestr": "|u1", "data": (base, False), "version": 2}

    memory = Memory()
    memory.owner = cache
    raw = torch.as_tensor(memory, device=DEVICE)
    b, kvh, d = case["block"], case["kv_heads"], case["dim"]
    if not case["q8"]:
        return raw.view(torch.float32).as_strided((blocks, layers, 2, b, kvh * d),
                                                  (stride // 4, 2 * b * kvh * d, b * kvh * d, kvh * d, 1))
    head = -(-(b * d + b * (d // 32) * 2) // 16) * 16
    ints = raw.view(torch.int8).as_strided((blocks, layers, 2, kvh, b, d),
                                           (stride, 2 * kvh * head, kvh * head, head, d, 1))
    h = raw.view(torch.float16)
    scales = h.as_strided((blocks, layers, 2, kvh, b, d // 32),
                          (stride // 2, kvh * head, kvh * head // 2, head // 2, d // 32, 1), b * d // 2)
    return ints, scales


# ------------------------------------------------------------------ trees

def _forest(st, case):
    """The trees as a program keeps them: packed parents, and padded to the
    largest the node rows, the ancestors (each node its own among them) and the parents."""
    trees = _trees(case)
    n, most = len(trees), max(len(t) for t in trees)
    st.nodes = np.array([len(t) for t in trees], dtype=np.uintp)
    st.parents = np.concatenate([np.array(t, np.int32) for t in trees])
    first = np.concatenate([[0], np.cumsum(st.nodes)[:-1]]).astype(np.int64)
    anc = np.zeros((n, most, most), bool)
    par = np.full((n, most), -2, np.int64)
    for i, t in enumerate(trees):
        for j, p in enumerate(t):
            if p >= 0:
                anc[i, j] = anc[i, p]
            anc[i, j, j] = True
        par[i, :len(t)] = t
    flat = np.concatenate([i * most + np.arange(len(t)) for i, t in enumerate(trees)])
    rows = np.minimum(first[:, None] + np.arange(most), len(st.parents) - 1)
    up = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(DEVICE)  # noqa: E731
    st.most, st.anc, st.par, st.flat, st.rows, st.first = most, up(anc), up(par), up(flat), up(rows), up(first)
    st.depth = max(max(_depths(t)) for t in trees)


def _texts(st, case, seed):
    """Logits as a bf16 model gives them (ties among them), tokens of a drafter
    that agrees with the model's choice now and then, and the token each root has to be."""
    total = len(st.parents)
    v = case["vocab"]
    st.logits = (3 * torch.randn(total, v, generator=_gen(seed, "logits"), device=DEVICE)).bfloat16().float()
    best = _argmax(st.logits)
    guess = torch.randint(0, v, (total,), generator=_gen(seed, "tokens"), device=DEVICE)
    agree = torch.rand(total, generator=_gen(seed, "agree"), device=DEVICE) < case["agree"]
    parent = torch.from_numpy(st.parents.astype(np.int64)).to(DEVICE)
    tree = torch.repeat_interleave(torch.arange(case["n"], device=DEVICE), torch.from_numpy(st.nodes.astype(np.int64)).to(DEVICE))
    want = best[(st.first[tree] + parent).clamp(min=0)]
    tokens = torch.where(agree & (parent >= 0), want, guess)
    first = tokens[st.first]
    miss = torch.rand(case["n"], generator=_gen(seed, "miss"), device=DEVICE) < 0.1
    st.expected = torch.where(miss, torch.randint(0, v, (case["n"],), generator=_gen(seed, "other"), device=DEVICE), first).int()
    st.tokens = tokens.int()
    st.path = torch.empty(case["n"], st.depth, dtype=torch.int32, device=DEVICE)
    st.accepted = torch.empty(case["n"], dtype=torch.int32, device=DEVICE)
    st.next = torch.empty(case["n"], dtype=torch.int32, device=DEVICE)


def _argmax(x):
    """The lowest index of each row's maximum."""
    top = x.amax(-1, keepdim=True)
    at = torch.arange(x.shape[-1], device=x.device)
    return torch.where(x == top, at, x.shape[-1]).amin(-1)


# -------------------------------------------------------------- the calls

def prepare(case, seed):
    kind = case["kind"]
    st = _State()
    st.case, st.kind = case, kind
    layers = st.layers = case.get("layers", 1)
    if kind == "accept":
        _forest(st, case)
        _texts(st, case, seed)
        if own:
            from tvara_amd import attention, kv

            # acceptance needs the trees alone: the sequences may be empty
            st.cache = kv.PagedCache(1, 1, 64, 16, 1)
            st.seqs = np.array([st.cache.create_sequence() for _ in range(case["n"])], dtype=np.uint64)
            st.plan = attention.TreePlan(st.cache, st.seqs, st.nodes, st.parents, 1, CONTEXT)
        return st
    lengths = _lengths(case)
    table = _tables(case)
    st.table = torch.from_numpy(table).to(DEVICE)
    if kind in ("slots", "write"):
        counts = _counts(case)
        if kind == "slots":  # the lengths are inputs: another seed has others in the same blocks
            r = random.Random(int(seed))
            counts = [r.randint(0, c) if case["n"] > 1 else c for c in counts]
            starts = [n + r.randint(0, m - c) for n, m, c in zip(lengths, _counts(case), counts)]
            if case["n"] == 1:
                starts = [r.randint(0, lengths[0])]
        else:
            starts = lengths
        st.starts = torch.tensor(starts, dtype=torch.int32, device=DEVICE)
        st.counts = torch.tensor(counts, dtype=torch.int32, device=DEVICE)
        stride = case.get("stride", 0)
        st.stride, st.cap = stride, max(1, case["n"] * stride if stride else sum(_counts(case)))
    if kind == "slots":
        st.offsets = torch.empty(case["n"] + 1, dtype=torch.int32, device=DEVICE)
        st.positions = torch.empty(st.cap, dtype=torch.int32, device=DEVICE)
        st.slots = torch.empty(st.cap, dtype=torch.int64, device=DEVICE)
        st.width = table.shape[1]
        st.tables = torch.empty(case["n"], st.width, dtype=torch.int32, device=DEVICE)
        if own:
            from tvara_amd import kv

            none = {"kv_heads": 1, "dim": 64, "q8": False}
            _cache(st, {**case, **none}, *(torch.zeros(sum(lengths), 64, device=DEVICE) for _ in "kv"), 1)
            st.cache.reserve(st.seqs, _counts(case))
            st.plan = kv.SlotPlan(st.cache, st.seqs)
        return st
    total = sum(lengths)
    k, v = (_kv_rows(case, seed, which, total, layers) for which in ("k", "v"))
    if kind == "write":
        counts = _counts(case)
        # accepted nodes in a batch of twice as many candidates, at fixed places a sequence
        most = max(1, max(counts))
        st.total = 2 * case["n"] * most
        kvw = case["kv_heads"] * case["dim"]
        st.nk, st.nv = (_kv_rows(case, seed, which, st.total, layers).reshape(st.total, layers, kvw) for which in ("tk", "tv"))
        if case["by_layer"]:
            st.nk, st.nv = (x.transpose(0, 1).contiguous() for x in (st.nk, st.nv))
        pos = st.starts[:, None].long() + torch.arange(most, device=DEVICE)
        blk = torch.gather(st.table, 1, (pos // case["block"]).clamp(max=st.table.shape[1] - 1))
        seen = torch.arange(most, device=DEVICE) < st.counts[:, None]
        st.slots = torch.where(seen, blk * case["block"] + pos % case["block"], -1).reshape(-1)
        pick = torch.rand(case["n"], 2 * most, generator=_gen(seed, "pick"), device=DEVICE).argsort(1)[:, :most].sort(1)[0]
        pick = pick + 2 * most * torch.arange(case["n"], device=DEVICE)[:, None]
        st.rows = torch.where(seen, pick, -1).int().reshape(-1)
        if own:
            from tvara_amd import kv

            _cache(st, case, k, v, layers)
            st.cache.reserve(st.seqs, counts)
            st.plan = kv.SlotPlan(st.cache, st.seqs)
            st.pool = _pool_of(st.cache, case, layers)
        else:
            st.pool = _pool(case, k, v, table, layers)
        return st
    _forest(st, case)
    nodes = len(st.parents)
    kvw, hidden = case["kv_heads"] * case["dim"], case["heads"] * case["dim"]
    st.q = 1.5 * torch.randn(layers, nodes, hidden, generator=_gen(seed, "q"), device=DEVICE)
    # a node's rows of all layers lie together, as the write of the accepted ones takes them
    st.nk, st.nv = (_kv_rows(case, seed, which, nodes, layers).reshape(nodes, layers, kvw) for which in ("tk", "tv"))
    st.out = torch.empty_like(st.q)
    st.starts = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
    st.longest = max(1, max(lengths))
    if kind == "step":
        _texts(st, case, seed)
        st.cap = case["n"] * st.depth
        st.positions = torch.empty(st.cap, dtype=torch.int32, device=DEVICE)
        st.slots = torch.empty(st.cap, dtype=torch.int64, device=DEVICE)
        st.offsets = torch.empty(case["n"] + 1, dtype=torch.int32, device=DEVICE)
    if own:
        from tvara_amd import attention

        _cache(st, case, k, v, layers, case["n"] * (st.depth // case["block"] + 2))
        if kind == "tree":
            st.plan = attention.TreePlan(st.cache, st.seqs, st.nodes, st.parents, case["heads"], CONTEXT,
                                         precision=case["precision"])
        else:
            st.room = np.full(case["n"], st.depth, np.uintp)
    else:
        st.pool = _pool(case, k, v, table, layers)
        if kind == "step":  # where the plain form puts a step's new rows, a slot for each
            room = {**case, "block": 1, "low": 1, "high": 1, "n": st.cap}
            none = torch.zeros(st.cap, layers * kvw, device=DEVICE)
            st.spare = _pool(room, none, none, np.arange(st.cap)[:, None], layers)
            st.place = torch.arange(st.cap, device=DEVICE)
    return st


def _plain_tree(st, layer):
    case = st.case
    heads, kvh, d, b = case["heads"], case["kv_heads"], case["dim"], case["block"]
    n, g, most = case["n"], heads // kvh, st.most
    q = st.q[layer].reshape(-1, kvh, g, d)[st.rows].permute(0, 2, 1, 3, 4).reshape(n, kvh, most * g, d)
    tail = [x[:, layer].reshape(-1, kvh, d)[st.rows] for x in (st.nk, st.nv)]
    length = st.longest
    pos = torch.arange(length, device=q.device)
    blk = st.table[:, pos // b].clamp(min=0)
    slot = (pos % b).expand(n, -1)
    kv = []
    for kind in (0, 1):
        if case["q8"]:
            ints, scales = st.pool
            x = _decode(ints[blk, layer, kind, :, slot], scales[blk, layer, kind, :, slot])
        else:
            x = st.pool[blk, layer, kind, slot].reshape(n, length, kvh, d)
        kv.append(torch.cat([x, tail[kind]], 1))
    seen = torch.cat([(pos < st.starts[:, None])[:, None].expand(-1, most, -1), st.anc], 2)
    s = torch.matmul(q, kv[0].permute(0, 2, 3, 1).contiguous()) / math.sqrt(d)
    s = s.masked_fill(~seen.repeat_interleave(g, 1)[:, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(p, kv[1].permute(0, 2, 1, 3).contiguous()) / p.sum(-1, keepdim=True)
    o = o.reshape(n, kvh, most, g, d).permute(0, 2, 1, 3, 4).reshape(n * most, heads * d)
    return o[st.flat]


def _plain_accept(st):
    """A node is confirmed where it is the lowest of its parent's children with
    the model's choice after the parent, and every node above it is."""
    n, most = st.par.shape
    best = _argmax(st.logits)[st.rows]
    up = torch.gather(best, 1, st.par.clamp(min=0))
    want = torch.where(st.par == -1, st.expected[:, None].long(), up)
    ok = (st.tokens.long()[st.rows] == want) & (st.par >= -1)
    at = torch.arange(most, device=ok.device)
    earlier = (st.par[:, :, None] == st.par[:, None, :]) & (at[None, :] < at[:, None]) & ok[:, None, :]
    ok &= ~earlier.any(2)
    on = ((st.anc & ~ok[:, None, :]).sum(2) == 0) & (st.par >= -1)
    count = on.sum(1)
    place = torch.where(on, at, most).sort(1)[0][:, :st.depth]
    path = torch.where(place < most, place + st.first[:, None], -1)
    last = torch.where(on, at, -1).amax(1)
    after = torch.gather(best, 1, last.clamp(min=0)[:, None])[:, 0]
    return path.int(), count.int(), torch.where(last >= 0, after, st.expected.long()).int()


def _plain_slots(st, starts, counts, stride, cap):
    n, b = st.table.shape[0], st.case["block"]
    end = torch.cumsum(counts.long(), 0)
    offsets = torch.cat([torch.zeros_like(end[:1]), end])
    t = torch.arange(cap, device=end.device)
    if stride:
        i, j = t // stride, t % stride
    else:
        i = torch.searchsorted(end, t, right=True)
        j = t - offsets[i.clamp(max=n - 1)]
    live = (i < n) & (j < counts.long()[i.clamp(max=n - 1)])
    i = i.clamp(max=n - 1)
    pos = starts.long()[i] + j
    blk = st.table[i, (pos // b).clamp(max=st.table.shape[1] - 1)]
    return offsets.int(), torch.where(live, pos, -1).int(), torch.where(live, blk * b + pos % b, -1)


def _plain_write(pool, case, slots, rows, nk, nv, layers):
    b, kvh, d = case["block"], case["kv_heads"], case["dim"]
    kv = torch.stack([nk, nv], 2)[rows.long().clamp(min=0)]
    live = torch.nonzero(slots >= 0)[:, 0]
    blk, slot = slots[live] // b, slots[live] % b
    if not case["q8"]:
        pool[blk, :, :, slot] = kv[live]
        return pool
    q, s = _encode(kv[live])
    pool[0][blk, :, :, :, slot] = q.reshape(-1, layers, 2, kvh, d)
    pool[1][blk, :, :, :, slot] = s.reshape(-1, layers, 2, kvh, d // 32)
    return pool


def _own(st):
    kind, case = st.kind, st.case
    if kind == "tree":
        st.plan.launch(0, st.q.data_ptr(), st.nk.data_ptr(), st.nv.data_ptr(), st.out.data_ptr())
        return st.out[0]
    if kind == "accept":
        st.plan.accept(st.tokens.data_ptr(), st.expected.data_ptr(), st.logits.data_ptr(), case["vocab"],
                       st.path.data_ptr(), st.depth, st.accepted.data_ptr(), st.next.data_ptr())
        return st.path, st.accepted, st.next
    if kind == "slots":
        st.plan.build(st.starts.data_ptr(), st.counts.data_ptr(), st.stride, st.cap, st.offsets.data_ptr(),
                      st.positions.data_ptr(), st.slots.data_ptr(), st.tables.data_ptr(), st.width)
        return st.offsets, st.positions, st.slots, st.tables
    kvw = case["kv_heads"] * case["dim"]
    if kind == "write":
        step = (kvw, st.total * kvw) if case["by_layer"] else (st.layers * kvw, kvw)
        st.plan.write(st.slots.data_ptr(), st.rows.data_ptr(), st.slots.numel(), st.nk.data_ptr(), st.nv.data_ptr(),
                      st.total, *step)
        return st.pool
    from tvara_amd import attention, kv

    st.cache.reserve(st.seqs, st.room)
    slots = kv.SlotPlan(st.cache, st.seqs)
    plan = attention.TreePlan(st.cache, st.seqs, st.nodes, st.parents, case["heads"], CONTEXT, visible=st.lengths,
                              precision=case["precision"])
    for layer in range(st.layers):
        plan.launch(layer, st.q[layer].data_ptr(), st.nk[:, layer].data_ptr(), st.nv[:, layer].data_ptr(),
                    st.out[layer].data_ptr(), row_stride=st.layers * kvw)
    plan.accept(st.tokens.data_ptr(), st.expected.data_ptr(), st.logits.data_ptr(), case["vocab"], st.path.data_ptr(),
                st.depth, st.accepted.data_ptr(), st.next.data_ptr())
    slots.build(st.starts.data_ptr(), st.accepted.data_ptr(), st.depth, st.cap, st.offsets.data_ptr(),
                st.positions.data_ptr(), st.slots.data_ptr())
    slots.write(st.slots.data_ptr(), st.path.data_ptr(), st.cap, st.nk.data_ptr(), st.nv.data_ptr(), len(st.parents),
                st.layers * kvw, kvw)
    st.cache.truncate_batch(st.seqs, st.lengths)
    return st.out, st.path, st.accepted, st.next, st.offsets, st.positions


def run(st):
    if own:
        return _own(st)
    kind, case = st.kind, st.case
    if kind == "tree":
        return _plain_tree(st, 0)
    if kind == "accept":
        return _plain_accept(st)
    if kind == "slots":
        return (*_plain_slots(st, st.starts, st.counts, st.stride, st.cap), st.table.int())
    nk, nv = (x.transpose(0, 1) if case.get("by_layer") else x for x in (st.nk, st.nv))
    if kind == "write":
        return _plain_write(st.pool, case, st.slots, st.rows, nk, nv, st.layers)
    out = torch.stack([_plain_tree(st, layer) for layer in range(st.layers)])
    path, count, after = _plain_accept(st)
    offsets, positions, _ = _plain_slots(st, st.starts, count, st.depth, st.cap)
    slots = torch.where(positions >= 0, st.place, -1)
    _plain_write(st.spare, {**case, "block": 1}, slots, path.reshape(-1), nk, nv, st.layers)
    return out, path, count, after, offsets, positions


# ------------------------------------------------------------ in 64 bits

def _held(x, q8):
    """What the cache holds of f32 rows, as float64."""
    if not q8:
        return x.double()
    g = x.reshape(x.shape[0], -1, 32)
    top = g.abs().amax(2, keepdim=True).double() / 127
    ints = torch.where(top > 0, (g.double() / top.float().double().clamp(min=1e-300)).float(), torch.zeros_like(g))
    return (torch.round(ints).clamp(-127, 127).double() * top.half().double()).reshape(x.shape)


def _exact_tree(case, seed):
    lengths, trees, layers = _lengths(case), _trees(case), case.get("layers", 1)
    heads, kvh, d = case["heads"], case["kv_heads"], case["dim"]
    k, v = (_kv_rows(case, seed, w, sum(lengths), layers) for w in ("k", "v"))
    nodes = sum(len(t) for t in trees)
    tk, tv = (_kv_rows(case, seed, w, nodes, layers) for w in ("tk", "tv"))
    q = 1.5 * torch.randn(layers, nodes, heads * d, generator=_gen(seed, "q"), device=DEVICE)
    out = torch.empty(q.shape, dtype=torch.float64, device=DEVICE)
    for layer in range(layers):
        cols = slice(layer * kvh * d, (layer + 1) * kvh * d)
        c0 = r0 = 0
        for n, parents in zip(lengths, trees):
            t = len(parents)
            kk, vv = (torch.cat([_held(x[c0:c0 + n, cols], case["q8"]), y[r0:r0 + t, cols].double()])
                      .reshape(n + t, kvh, d) for x, y in ((k, tk), (v, tv)))
            for h in range(kvh):
                g = heads // kvh
                rows = q[layer, r0:r0 + t].double().reshape(t, heads, d)[:, h * g:(h + 1) * g]
                s = torch.tensordot(rows, kk[:, h], ([2], [1])) / math.sqrt(d)
                mask = torch.ones(t, n + t, dtype=torch.bool)
                mask[:, n:] = False
                for j in range(t):
                    a = j
                    while a >= 0:
                        mask[j, n + a] = True
                        a = parents[a]
                s.masked_fill_(~mask.to(DEVICE)[:, None], -math.inf)
                o = torch.tensordot(torch.softmax(s, 2), vv[:, h], ([2], [0]))
                out[layer, r0:r0 + t].view(t, heads, d)[:, h * g:(h + 1) * g] = o
            c0, r0 = c0 + n, r0 + t
    return out


def exact(case, seed):
    """run()'s answer in 64 bits; whole numbers have none."""
    kind = case["kind"]
    if kind in ("accept", "slots"):
        return None
    if kind == "tree":
        return _exact_tree(case, seed)[0]
    if kind == "step":
        return _exact_tree(case, seed), None, None, None, None, None
    lengths, counts, layers, b = _lengths(case), _counts(case), case["layers"], case["block"]
    table = _tables(case)
    kvh, d = case["kv_heads"], case["dim"]
    k, v = (_kv_rows(case, seed, w, sum(lengths), layers) for w in ("k", "v"))
    most = max(1, max(counts))
    new = [_kv_rows(case, seed, w, 2 * case["n"] * most, layers) for w in ("tk", "tv")]
    pick = torch.rand(case["n"], 2 * most, generator=_gen(seed, "pick"), device=DEVICE).argsort(1)[:, :most].sort(1)[0].cpu()
    blocks = int(table.max()) + 1
    full = torch.zeros(blocks, layers, 2, b, kvh * d, dtype=torch.float64, device=DEVICE)
    c0 = 0
    for i, n in enumerate(lengths):
        rows = pick[i, :counts[i]].to(DEVICE) + 2 * most * i
        for kind_at, (x, y) in enumerate(((k, new[0]), (v, new[1]))):
            all_rows = torch.cat([x[c0:c0 + n], y[rows]]).double().reshape(-1, layers, kvh * d)
            for lo in range(0, n + counts[i], b):
                part = all_rows[lo:lo + b]
                full[table[i, lo // b], :, kind_at, :part.shape[0]] = part.transpose(0, 1)
        c0 += n
    if not case["q8"]:
        return full
    scales = full.reshape(blocks, layers, 2, b, kvh, d // 32, 32).abs().amax(-1) / 127
    return None, scales.permute(0, 1, 2, 4, 3, 5)
