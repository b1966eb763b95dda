"""Entry points of scored attention, rotation into the cache, reading back and sampling:
closed handles, sizes and arguments that are refused, and the ranges of keys (no device
calls: CPU only)."""

import numpy as np
import pytest

from tvara_amd import _capi, attention, sampling


def test_closed_handles_are_refused():
    lib = _capi.lib()
    for rc in (lib.tvara_score_plan_launch(None, 0, None, None, None), lib.tvara_score_plan_check(None),
               lib.tvara_attn_score(None, None, 0, 0, 1, 1, None, None, None, None, 0.0, 0.0, None, None, None, 0),
               lib.tvara_slot_plan_rotate(None, None, 0, 0, 1, None, 0, None, None, 0, None, None, 0, 0, None, None, 0.0, None,
                                          None, None),
               lib.tvara_slot_plan_read(None, None, 0, 0, 0, None, None, 0, 0, None),
               lib.tvara_sample_plan_launch(None, 1, None, 0, None, None, None, None, None, None, None, None),
               lib.tvara_sample_plan_check(None)):
        assert rc == _capi.INVALID
    assert not lib.tvara_score_plan_create(None, None, 0, 1, 1, None, None, None, None, 0.0, 0.0, None)
    assert lib.tvara_last_status() == _capi.INVALID
    lib.tvara_score_plan_destroy(None)
    lib.tvara_sample_plan_destroy(None)


def test_closed_model_is_refused():
    lib = _capi.lib()
    assert lib.tvara_sequences_sample(None, None, None, 0, None, None, None, None, None, None, None) == -1
    assert lib.tvara_last_error() == b"invalid batch buffers"


@pytest.mark.parametrize("rows,vocab", [(0, 5), (5, 0), (65536, 5), (1 << 40, 5), (1, 1 << 30), (65535, 1 << 18)])
def test_sample_plans_too_large_or_empty(rows, vocab):
    with pytest.raises(_capi.InvalidArgument):
        sampling.SamplePlan(rows, vocab)


@pytest.mark.parametrize("how", [dict(uniforms=[0.5]), dict(uniforms=0.5), dict(top_k=[1, 2, 3]), dict(top_k=1.5), dict(top_k=-1),
                                 dict(top_k=[1, 1 << 31]), dict(temperature=[1.0]), dict(top_p=np.ones((2, 1)))])
def test_sampling_arguments_of_other_lengths(how):
    with pytest.raises(_capi.InvalidArgument):
        sampling.sample_batch(np.zeros((2, 4), np.float32), **{"uniforms": [0.5, 0.5], **how})
    with pytest.raises(_capi.InvalidArgument):
        sampling.sample_batch(np.zeros(4, np.float32), [0.5])


def test_no_rows_to_sample():
    tokens, chances = sampling.sample_batch(np.zeros((0, 4), np.float32), [])
    assert tokens.size == chances.size == 0 and tokens.dtype == np.uint32


def by_hand(starts, counts, window, prefix, document):
    first, end, r = [], [], 0
    for i, (s, c) in enumerate(zip(starts, counts)):
        for p in range(s, s + c):
            lo, hi = 0, p + 1
            if window is not None:
                lo = max(lo, p + 1 - window)
            if document is not None:
                lo = max(lo, document[r])
            if prefix is not None and p < prefix[i]:
                hi = prefix[i]
            first.append(lo)
            end.append(hi)
            r += 1
    return first, end


@pytest.mark.parametrize("window", [None, 1, 3, 1 << 70])
@pytest.mark.parametrize("prefix", [None, [0, 4, 2, 9]])
@pytest.mark.parametrize("documents", [False, True])
def test_ranges(window, prefix, documents):
    starts, counts = [0, 2, 7, 5], [3, 4, 0, 1]
    document = [0, 1, 1, 0, 3, 3, 5, 2] if documents else None
    first, end = attention.visible_ranges(starts, counts, window, prefix, document)
    want = by_hand(starts, counts, window, prefix, document)
    assert first.tolist() == want[0] and end.tolist() == want[1]
    assert first.dtype == end.dtype == np.uintp


def test_ranges_of_nothing():
    first, end = attention.visible_ranges([], [])
    assert first.size == end.size == 0
    first, end = attention.visible_ranges([4, 9], [0, 0], window=2)
    assert first.size == end.size == 0


@pytest.mark.parametrize("how", [dict(starts=[1]), dict(counts=[1.5, 1]), dict(starts=[-1, 0]), dict(window=0), dict(document=[0]),
                                 dict(document=[0, -1.5]), dict(prefix=[0.5, 1])])
def test_ranges_refused(how):
    with pytest.raises(_capi.InvalidArgument):
        attention.visible_ranges(**{"starts": [0, 0], "counts": [1, 1], **how})


@pytest.mark.parametrize("how", [dict(starts=[0]), dict(counts=[1, 1, 1]), dict(counts=[1, -1]), dict(first=[0]), dict(end=[1, 1, 1]),
                                 dict(first=[0.5, 0]), dict(end=[-1, 1]), dict(slopes=[1.0])])
def test_scored_arguments_of_other_lengths(how):
    given = {"seqs": [1, 2], "starts": [0, 0], "counts": [1, 1], "heads": 4, "first": None, "end": None, "slopes": None, **how}
    with pytest.raises(_capi.InvalidArgument):
        attention._scored(**given)
