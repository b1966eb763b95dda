"""The next token of rows of logits on the GPU (tvara_sample_plan_*): temperature,
top-k, top-p and min-p from given random numbers, as the reference's host
samples (python/tvara/native.py:301-334) without their penalties and masks
(a masked token's logit is -inf).
"""

from __future__ import annotations

import ctypes as C

import numpy as np

from . import _capi
from ._capi import InvalidArgument


def f32_below_one(uniforms):
    """Random numbers in f32: those below 1 in a wider type, the last 2^-25 before it
    too, stay below 1."""
    given = np.asarray(uniforms)
    u = given.astype(np.float32)
    return np.where((u == 1) & (given < 1), np.nextafter(np.float32(1), np.float32(0)), u)


class SamplePlan:
    """Workspace for up to ``rows`` rows of ``vocab`` logits."""

    def __init__(self, rows, vocab):
        self.lib = _capi.lib()
        self.rows, self.vocab = rows, vocab
        self.h = self.lib.tvara_sample_plan_create(rows, vocab)
        if not self.h:
            _capi.raise_last()

    def launch(self, logits_ptr, uniforms_ptr, tokens_ptr, probability_ptr=None, temperature_ptr=None, top_k_ptr=None,
               top_p_ptr=None, min_p_ptr=None, rows=None, logits_stride=0, stream=None):
        """Asynchronous over device pointers (ints): f32 logits, uniforms and
        parameters, int32 top_k (None: temperature 1, everything kept), uint32
        tokens and f32 probabilities of the first ``rows`` rows (None: all)."""
        _capi.check(self.lib.tvara_sample_plan_launch(self.h, self.rows if rows is None else rows, logits_ptr, logits_stride,
                                                      uniforms_ptr, temperature_ptr, top_k_ptr, top_p_ptr, min_p_ptr,
                                                      tokens_ptr, probability_ptr, stream))

    def check(self):
        _capi.check(self.lib.tvara_sample_plan_check(self.h))

    def close(self):
        if getattr(self, "h", None):
            self.lib.tvara_sample_plan_destroy(self.h)
            self.h = None

    def __del__(self):
        self.close()


def sample_batch(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Tokens and probabilities of rows of host logits [n, vocab] (synchronous);
    the parameters one for all rows or one for each."""
    from . import hip

    logits = np.ascontiguousarray(logits, dtype=np.float32)
    if logits.ndim != 2:
        raise InvalidArgument("logits are rows of a vocabulary")
    n, vocab = logits.shape
    if not n:
        return np.zeros(0, np.uint32), np.zeros(0, np.float32)

    def each(values, dtype, what):
        values = np.asarray(values)
        if values.ndim and values.shape != (n,):
            raise InvalidArgument(f"one {what} for all rows or for each")
        if dtype is np.int32 and (values.dtype.kind not in "iu" or (values < 0).any() or (values > 2**31 - 1).any()):
            raise InvalidArgument(f"{what} is a whole number from 0")
        return np.ascontiguousarray(np.broadcast_to(values.astype(dtype), (n,)))

    if np.shape(uniforms) != (n,):
        raise InvalidArgument("one random number for each row")
    given = [each(x, t, what) for x, t, what in ((f32_below_one(uniforms), np.float32, "random number"),
                                                 (temperature, np.float32, "temperature"), (top_k, np.int32, "top_k"),
                                                 (top_p, np.float32, "top_p"), (min_p, np.float32, "min_p"))]
    x, *given = (hip.DeviceArray.from_numpy(a) for a in (logits, *given))
    tokens, chances = hip.DeviceArray((n,), np.uint32), hip.DeviceArray((n,), np.float32)
    plan = SamplePlan(n, vocab)
    u, t, k, p, m = (d.ptr for d in given)
    plan.launch(x.ptr, u, tokens.ptr, chances.ptr, t, k, p, m)
    plan.check()
    return tokens.numpy(), chances.numpy()
