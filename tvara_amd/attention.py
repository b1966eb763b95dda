"""Paged attention over a device ``PagedCache`` (libtvara_capi.so).

* ``fused_paged_attention`` -- attention.hpp:57-83, one query row;
* ``decode_batch`` -- the same for many sequences in one launch;
* ``fused_prompt_attention`` / ``prefill_batch`` -- attention.hpp:85-89, a
  causal chunk over cached positions, in f32 (reference semantics) or on bf16
  MFMA tiles;
* ``DecodePlan`` -- resident block tables for repeated device launches;
* ``TreePlan`` / ``tree_batch`` -- trees of drafted tokens over cached
  sequences: their attention and their greedy acceptance;
* ``ScorePlan`` / ``score_batch`` -- attention with capped or biased scores,
  each row within a range of keys of its own (``visible_ranges``).
"""

from __future__ import annotations

import ctypes as C

import numpy as np

from . import _capi
from ._capi import InvalidArgument

_fp = C.POINTER(C.c_float)
_sz = C.c_size_t
_NO_CAP = (1 << 64) - 1
_PRECISION = {"f32": _capi.ATTN_F32, "bf16": _capi.ATTN_BF16, "f32x3": _capi.ATTN_F32X3}


def _f32(a):
    return np.ascontiguousarray(a, dtype=np.float32)


def _ptr(a):
    return a.ctypes.data_as(_fp) if a is not None else None


def decode_batch(cache, q, seqs, layer, heads, context, tail_keys=None, tail_values=None, visible=None):
    """fused_paged_attention for every listed sequence: q [n, heads*head_dim]."""
    seqs = np.ascontiguousarray(seqs, dtype=np.uint64).reshape(-1)
    n = seqs.size
    hidden = heads * cache.head_dim
    q = _f32(q).reshape(n, hidden) if n else _f32(q)
    tk = _f32(tail_keys).reshape(n, cache.kv_width) if tail_keys is not None else None
    tv = _f32(tail_values).reshape(n, cache.kv_width) if tail_values is not None else None
    vis = None
    if visible is not None:
        vis = np.ascontiguousarray(np.broadcast_to(np.asarray(visible, dtype=np.uint64), (n,)))
    out = np.empty((max(n, 1), hidden), np.float32)
    rc = cache.lib.tvara_attn_decode(cache.h, seqs.ctypes.data_as(C.POINTER(C.c_uint64)), n, layer, heads, context,
                                     _ptr(q), _ptr(tk), _ptr(tv),
                                     vis.ctypes.data_as(C.POINTER(_sz)) if vis is not None else None, _ptr(out), 0)
    _capi.check(rc)
    return out[:n]


def fused_paged_attention(q, cache, sequence, layer, heads, context, tail_key=None, tail_value=None, visible=None):
    """fused_paged_attention (attention.hpp:57-83): one row of heads*head_dim."""
    tk = None if tail_key is None else _f32(tail_key).reshape(1, -1)
    tv = None if tail_value is None else _f32(tail_value).reshape(1, -1)
    vis = None if visible is None else [visible]
    return decode_batch(cache, _f32(q).reshape(1, -1), [sequence], layer, heads, context, tk, tv, vis)[0]


def prefill_batch(cache, queries, seqs, starts, counts, layer, heads, context, precision="f32"):
    """fused_prompt_attention for several sequences; queries packed by sequence."""
    seqs = np.ascontiguousarray(seqs, dtype=np.uint64).reshape(-1)
    starts = np.ascontiguousarray(starts, dtype=np.uint64).reshape(-1)
    counts = np.ascontiguousarray(counts, dtype=np.uint64).reshape(-1)
    if precision not in _PRECISION:
        raise InvalidArgument("unknown attention precision")
    hidden = heads * cache.head_dim
    rows = int(counts.sum())
    q = _f32(queries).reshape(rows, hidden)
    out = np.empty((max(rows, 1), hidden), np.float32)
    rc = cache.lib.tvara_attn_prefill(cache.h, seqs.ctypes.data_as(C.POINTER(C.c_uint64)), seqs.size, layer, heads,
                                      context, starts.ctypes.data_as(C.POINTER(_sz)),
                                      counts.ctypes.data_as(C.POINTER(_sz)), _ptr(q), _ptr(out),
                                      _PRECISION[precision], 0)
    _capi.check(rc)
    return out[:rows]


def fused_prompt_attention(queries, cache, sequence, layer, start, count, heads, context, precision="f32"):
    """fused_prompt_attention (attention.hpp:85-89): rows start .. start+count-1."""
    return prefill_batch(cache, queries, [sequence], [start], [count], layer, heads, context, precision).reshape(-1)


def prefill_batch_device(cache, q_ptr, out_ptr, seqs, starts, counts, layer, heads, context, precision="bf16"):
    """prefill_batch over device buffers (synchronous)."""
    seqs = np.ascontiguousarray(seqs, dtype=np.uint64).reshape(-1)
    starts = np.ascontiguousarray(starts, dtype=np.uint64).reshape(-1)
    counts = np.ascontiguousarray(counts, dtype=np.uint64).reshape(-1)
    rc = cache.lib.tvara_attn_prefill(cache.h, seqs.ctypes.data_as(C.POINTER(C.c_uint64)), seqs.size, layer, heads,
                                      context, starts.ctypes.data_as(C.POINTER(_sz)),
                                      counts.ctypes.data_as(C.POINTER(_sz)), C.cast(q_ptr, _fp),
                                      C.cast(out_ptr, _fp), _PRECISION[precision], 1)
    _capi.check(rc)


class DecodePlan:
    """Resident block tables for one batch of sequences (tvara_attn_plan_*)."""

    def __init__(self, cache, seqs, heads, context, visible=None, with_tail=False):
        self.cache = cache
        self.lib = cache.lib
        seqs = np.ascontiguousarray(seqs, dtype=np.uint64).reshape(-1)
        vis = None
        if visible is not None:
            vis = np.ascontiguousarray(np.broadcast_to(np.asarray(visible, dtype=np.uint64), seqs.shape))
        self.h = self.lib.tvara_attn_plan_create(cache.h, seqs.ctypes.data_as(C.POINTER(C.c_uint64)), seqs.size, heads,
                                                 context, vis.ctypes.data_as(C.POINTER(_sz)) if vis is not None else None,
                                                 int(with_tail))
        if not self.h:
            _capi.raise_last()
        split, items, kv = _sz(), _sz(), _sz()
        _capi.check(self.lib.tvara_attn_plan_info(self.h, C.byref(split), C.byref(items), C.byref(kv)))
        self.split_tokens, self.items, self.kv_bytes = split.value, items.value, kv.value

    def launch(self, layer, q_ptr, out_ptr, tail_k_ptr=None, tail_v_ptr=None, stream=None):
        """Asynchronous launch over device pointers (ints)."""
        _capi.check(self.lib.tvara_attn_plan_decode(self.h, layer, q_ptr, tail_k_ptr, tail_v_ptr, out_ptr, stream))

    def check(self):
        _capi.check(self.lib.tvara_attn_plan_check(self.h))

    def close(self):
        if getattr(self, "h", None):
            self.lib.tvara_attn_plan_destroy(self.h)
            self.h = None

    def __del__(self):
        self.close()


class PrefillPlan:
    """Resident block tables for one chunked-prefill batch (tvara_prefill_plan_*):
    sequence i attends its rows starts[i] .. starts[i] + counts[i] - 1."""

    def __init__(self, cache, seqs, starts, counts, heads, context, precision="bf16"):
        self.cache = cache
        self.lib = cache.lib
        seqs = np.ascontiguousarray(seqs, dtype=np.uint64).reshape(-1)
        starts = np.ascontiguousarray(starts, dtype=np.uint64).reshape(-1)
        counts = np.ascontiguousarray(counts, dtype=np.uint64).reshape(-1)
        if not (seqs.size == starts.size == counts.size):
            raise ValueError("seqs, starts and counts differ in length")
        self.rows = int(counts.sum())
        self.h = self.lib.tvara_prefill_plan_create(cache.h, seqs.ctypes.data_as(C.POINTER(C.c_uint64)), seqs.size,
                                                    heads, context, starts.ctypes.data_as(C.POINTER(_sz)),
                                                    counts.ctypes.data_as(C.POINTER(_sz)), _PRECISION[precision])
        if not self.h:
            _capi.raise_last()

    def launch(self, layer, q_ptr, out_ptr, stream=None):
        """Asynchronous launch over device pointers (ints)."""
        _capi.check(self.lib.tvara_prefill_plan_launch(self.h, layer, q_ptr, out_ptr, stream))

    def check(self):
        _capi.check(self.lib.tvara_prefill_plan_check(self.h))

    def close(self):
        if getattr(self, "h", None):
            self.lib.tvara_prefill_plan_destroy(self.h)
            self.h = None

    def __del__(self):
        self.close()


def _whole(values, dtype, what):
    """values as an array of dtype, none of which it changes."""
    given = np.asarray(values)
    with np.errstate(invalid="ignore"):
        out = np.ascontiguousarray(given.astype(dtype))
    if not (given == out).all():
        raise InvalidArgument(f"{what} are not whole numbers of their range")
    return out


def _trees(seqs, nodes, parents, visible):
    seqs = np.ascontiguousarray(seqs, dtype=np.uint64).reshape(-1)
    nodes = _whole(nodes, np.uintp, "nodes").reshape(-1)
    parents = _whole(parents, np.int32, "parents").reshape(-1)
    if nodes.size != seqs.size or int(nodes.sum()) != parents.size:
        raise InvalidArgument("sequences, nodes and parents differ in length")
    if visible is not None:
        visible = np.ascontiguousarray(np.broadcast_to(_whole(visible, np.uintp, "visible lengths"), seqs.shape))
    vp = visible.ctypes.data_as(C.POINTER(_sz)) if visible is not None else None
    keep = (seqs, nodes, parents, visible)
    return keep, (seqs.ctypes.data_as(C.POINTER(C.c_uint64)), nodes.ctypes.data_as(C.POINTER(_sz)),
                  parents.ctypes.data_as(C.POINTER(C.c_int32)), vp)


def tree_batch(cache, q, seqs, nodes, parents, keys, values, layer, heads, context, visible=None, precision="f32"):
    """Attention of trees of drafted tokens (tvara_attn_tree): tree i hangs on
    seqs[i] and has nodes[i] of the packed nodes, parents (-1: a root) within
    its tree; q [nodes, heads * head_dim], keys and values [nodes, kv_width]."""
    if precision not in _PRECISION:
        raise InvalidArgument("unknown attention precision")
    (seqs, nodes, parents, visible), (sp, np_, pp, vp) = _trees(seqs, nodes, parents, visible)
    rows, hidden = parents.size, heads * cache.head_dim
    q = _f32(q).reshape(rows, hidden)
    k, v = _f32(keys).reshape(rows, cache.kv_width), _f32(values).reshape(rows, cache.kv_width)
    out = np.empty((max(rows, 1), hidden), np.float32)
    _capi.check(cache.lib.tvara_attn_tree(cache.h, sp, seqs.size, layer, heads, context, vp, np_, pp, _ptr(q), _ptr(k),
                                          _ptr(v), _ptr(out), _PRECISION[precision], 0))
    return out[:rows]


class TreePlan:
    """Resident trees of drafted tokens over cached sequences (tvara_tree_plan_*)."""

    def __init__(self, cache, seqs, nodes, parents, heads, context, visible=None, precision="f32"):
        if precision not in _PRECISION:
            raise InvalidArgument("unknown attention precision")
        self.cache = cache
        self.lib = cache.lib
        (seqs, nodes, parents, visible), (sp, np_, pp, vp) = _trees(seqs, nodes, parents, visible)
        self.rows = parents.size
        self.h = self.lib.tvara_tree_plan_create(cache.h, sp, seqs.size, heads, context, vp, np_, pp,
                                                 _PRECISION[precision])
        if not self.h:
            _capi.raise_last()

    def launch(self, layer, q_ptr, keys_ptr, values_ptr, out_ptr, row_stride=0, stream=None):
        """Asynchronous attention over device pointers (ints); K/V rows are
        row_stride floats apart (0: kv_width)."""
        _capi.check(self.lib.tvara_tree_plan_launch(self.h, layer, q_ptr, keys_ptr, values_ptr, row_stride, out_ptr,
                                                    stream))

    def accept(self, tokens_ptr, first_ptr, logits_ptr, vocab, path_ptr, path_stride, accepted_ptr, next_ptr,
               logits_stride=0, stream=None):
        """Asynchronous greedy acceptance over device pointers (ints)."""
        _capi.check(self.lib.tvara_tree_plan_accept(self.h, tokens_ptr, first_ptr, logits_ptr, vocab, logits_stride,
                                                    path_ptr, path_stride, accepted_ptr, next_ptr, stream))

    def check(self):
        _capi.check(self.lib.tvara_tree_plan_check(self.h))

    def close(self):
        if getattr(self, "h", None):
            self.lib.tvara_tree_plan_destroy(self.h)
            self.h = None

    def __del__(self):
        self.close()


def visible_ranges(starts, counts, window=None, prefix=None, document=None):
    """(first, end) of the keys that each row sees, for ScorePlan: the text up to
    itself and, where given, of that

    * window: itself and the window - 1 tokens before it;
    * prefix (one for each sequence): rows of a sequence's first prefix tokens
      see all of those;
    * document (one for each row): no token before the first of its document.
    """
    starts = _whole(starts, np.uintp, "starts").reshape(-1)
    counts = _whole(counts, np.uintp, "counts").reshape(-1)
    if starts.size != counts.size:
        raise InvalidArgument("starts and counts differ in length")
    seq = np.repeat(np.arange(counts.size), counts.astype(np.int64))
    before = np.concatenate([[0], np.cumsum(counts)[:-1]]).astype(np.int64) if counts.size else np.zeros(0, np.int64)
    pos = starts.astype(np.int64)[seq] + np.arange(seq.size) - before[seq]
    first, end = np.zeros(seq.size, np.int64), pos + 1
    if window is not None:
        if window < 1:
            raise InvalidArgument("a window has at least the row itself")
        first = np.maximum(first, end - int(min(window, 1 << 62)))
    if document is not None:
        document = _whole(document, np.int64, "documents").reshape(-1)
        if document.size != seq.size:
            raise InvalidArgument("one document start for each row")
        first = np.maximum(first, document)
    if prefix is not None:
        whole = np.broadcast_to(_whole(prefix, np.int64, "prefixes"), counts.shape)[seq]
        end = np.where(pos < whole, whole, end)
    return first.astype(np.uintp), end.astype(np.uintp)


def _scored(seqs, starts, counts, heads, first, end, slopes):
    seqs = np.ascontiguousarray(seqs, dtype=np.uint64).reshape(-1)
    starts = _whole(starts, np.uintp, "starts").reshape(-1)
    counts = _whole(counts, np.uintp, "counts").reshape(-1)
    if not seqs.size == starts.size == counts.size:
        raise InvalidArgument("sequences, starts and counts differ in length")
    rows = int(counts.sum())
    if first is not None:
        first = _whole(first, np.uintp, "first keys").reshape(-1)
    if end is not None:
        end = _whole(end, np.uintp, "ends of keys").reshape(-1)
    if any(x is not None and x.size != rows for x in (first, end)):
        raise InvalidArgument("one range of keys for each row")
    if slopes is not None:
        slopes = _f32(slopes).reshape(-1)
        if slopes.size != heads:
            raise InvalidArgument("one slope for each query head")

    def sizes(x):
        return x.ctypes.data_as(C.POINTER(_sz)) if x is not None else None

    keep = (seqs, starts, counts, first, end, slopes)
    return rows, keep, (seqs.ctypes.data_as(C.POINTER(C.c_uint64)), sizes(starts), sizes(counts), sizes(first), sizes(end),
                        _ptr(slopes))


def _score_call(lib, name, precision):
    """A call of scored attention: f32x3 (long chunks by fp16 parts) or f32 throughout."""
    if precision not in ("f32", "f32x3"):
        raise InvalidArgument("scored attention is f32x3 or f32")
    return getattr(lib, name + ("_f32" if precision == "f32" else ""))


def score_batch(cache, q, seqs, starts, counts, layer, heads, context, first=None, end=None, scale=None, cap=0.0,
                slopes=None, precision="f32x3"):
    """Scored attention (tvara_attn_score) of the cached rows starts[i] ..
    starts[i] + counts[i] - 1 of seqs[i], packed: q [rows, heads * head_dim]."""
    call = _score_call(cache.lib, "tvara_attn_score", precision)
    rows, keep, (sp, st, ct, fp, ep, bp) = _scored(seqs, starts, counts, heads, first, end, slopes)
    hidden = heads * cache.head_dim
    q = _f32(q).reshape(rows, hidden)
    out = np.empty((max(rows, 1), hidden), np.float32)
    _capi.check(call(cache.h, sp, keep[0].size, layer, heads, context, st, ct, fp, ep, scale or 0.0, cap, bp, _ptr(q),
                     _ptr(out), 0))
    return out[:rows]


class ScorePlan:
    """Resident rows of scored attention over cached sequences
    (tvara_score_plan_*): scores are scale * q.k, capped as cap * tanh(s / cap)
    where cap is above 0, less slopes[head] times the distance of key and row;
    row r sees the keys first[r] .. end[r] - 1 (None: from 0, to itself).  precision
    f32x3: chunks of many rows by fp16 parts, whose range tvara_capi.h states; f32:
    f32 products for all rows."""

    def __init__(self, cache, seqs, starts, counts, heads, context, first=None, end=None, scale=None, cap=0.0, slopes=None,
                 precision="f32x3"):
        create = _score_call(cache.lib, "tvara_score_plan_create", precision)
        self.cache = cache
        self.lib = cache.lib
        self.rows, keep, (sp, st, ct, fp, ep, bp) = _scored(seqs, starts, counts, heads, first, end, slopes)
        self.h = create(cache.h, sp, keep[0].size, heads, context, st, ct, fp, ep, scale or 0.0, cap, bp)
        if not self.h:
            _capi.raise_last()

    def launch(self, layer, q_ptr, out_ptr, stream=None):
        """Asynchronous attention over device pointers (ints)."""
        _capi.check(self.lib.tvara_score_plan_launch(self.h, layer, q_ptr, out_ptr, stream))

    def check(self):
        _capi.check(self.lib.tvara_score_plan_check(self.h))

    def close(self):
        if getattr(self, "h", None):
            self.lib.tvara_score_plan_destroy(self.h)
            self.h = None

    def __del__(self):
        self.close()


def profile_enable(on=True):
    _capi.check(_capi.lib().tvara_profile_enable(int(on)))


def profile_reset():
    _capi.check(_capi.lib().tvara_profile_reset())


def profile_read(kernel=None):
    ms, n = C.c_double(), _sz()
    _capi.check(_capi.lib().tvara_profile_read(kernel.encode() if kernel else None, C.byref(ms), C.byref(n)))
    return ms.value, n.value
