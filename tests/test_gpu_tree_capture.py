"""Captured launches of tree and slot plans: what a graph may and may not hold."""

import numpy as np
import pytest

import test_gpu_tree as tt
from tvara_amd import _capi, attention, hip
from tvara_amd.kv import SlotPlan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("what", ["attention", "write", "decode", "prefill"])
def test_replays_leave_blocks_handed_out_before(device, oracle, what):
    """A block that still waits for its zeros when a plan is made: a graph of the plan's
    launches does not clear it, however often it is replayed."""
    tt.say("tree captured, block handed out", what)
    b = tt.Batch(device, oracle, 4, 2, 64, [40], [tt.chain(3)], seed=2, spare=2)
    stream = hip.Stream()
    hip.synchronize()
    b.cache.set_stream(stream.h)
    h = b.cache.allocate()
    up = hip.DeviceArray.from_numpy
    with tt.hip_rows(b) as d:
        if what == "attention":
            plan = attention.TreePlan(b.cache, b.seqs, b.nodes, b.parents, 4, 1 << 20)
            launch = lambda: plan.launch(0, d.q.ptr, d.k.ptr, d.v.ptr, d.out.ptr, stream=stream.h)  # noqa: E731
        elif what == "decode":
            plan = attention.DecodePlan(b.cache, b.seqs, 4, 1 << 20)
            launch = lambda: plan.launch(0, d.q.ptr, d.out.ptr, stream=stream.h)  # noqa: E731
        elif what == "prefill":
            plan = attention.PrefillPlan(b.cache, b.seqs, [0], [3], 4, 1 << 20)
            launch = lambda: plan.launch(0, d.q.ptr, d.out.ptr, stream=stream.h)  # noqa: E731
        else:
            plan = SlotPlan(b.cache, b.seqs)
            slots = up(np.full(4, -1, np.int64))
            launch = lambda: plan.write(slots.ptr, None, 4, d.k.ptr, d.v.ptr, 3, b.w, b.w, stream=stream.h)  # noqa: E731
        graph = tt.Graph(stream.h, launch)
        assert not b.cache.block_data(h).any()
        for i in range(3):
            mine = np.full(b.cache.block_data(h).size, i + 1.0, np.float32)
            b.cache.block_write(h, 0, mine)
            graph.replay()
            plan.check()
            assert np.array_equal(b.cache.block_data(h), mine)
        if what == "attention":
            tt.agree(d.out.numpy()[: b.rows], b.want(), "f32")
        del graph
    hip.synchronize()
    b.cache.set_stream(None)


@pytest.mark.parametrize("own", [False, True])
def test_captures_on_another_stream_are_refused(device, oracle, own):
    """The cache's stream takes no part in such a capture: every launch is refused, the
    capture goes on, and so does eager work."""
    tt.say("captures on another stream", own)
    b = tt.Batch(device, oracle, 4, 2, 64, [40, 30], [tt.chain(3), [-1]], seed=2)
    streams = hip.Stream(), hip.Stream()
    hip.synchronize()
    b.cache.set_stream(streams[1].h if own else None)
    up, s = hip.DeviceArray.from_numpy, streams[0].h
    with tt.hip_rows(b) as d:
        tree, slots = attention.TreePlan(b.cache, b.seqs, b.nodes, b.parents, 4, 1 << 20), SlotPlan(b.cache, b.seqs)
        decode = attention.DecodePlan(b.cache, b.seqs, 4, 1 << 20)
        prefill = attention.PrefillPlan(b.cache, b.seqs, [0, 0], [2, 2], 4, 1 << 20, precision="f32")
        ints, words, logits = up(np.zeros(64, np.int32)), up(np.full(16, -1, np.int64)), up(np.zeros((4, 8), np.float32))
        calls = [lambda: tree.launch(0, d.q.ptr, d.k.ptr, d.v.ptr, d.out.ptr, stream=s),
                 lambda: tree.accept(ints.ptr, ints.ptr, logits.ptr, 8, ints.ptr + 64, 4, ints.ptr + 128, ints.ptr + 192, stream=s),
                 lambda: slots.build(ints.ptr, ints.ptr, 4, 8, slots_ptr=words.ptr, stream=s),
                 lambda: slots.write(words.ptr, None, 4, d.k.ptr, d.v.ptr, 4, b.w, b.w, stream=s),
                 lambda: decode.launch(0, d.q.ptr, d.out.ptr, stream=s),
                 lambda: prefill.launch(0, d.q.ptr, d.out.ptr, stream=s)]

        def body():
            for call in calls:
                with pytest.raises(_capi.InvalidArgument, match="captured on the cache's stream"):
                    call()

        graph = tt.Graph(s, body)
        for call in calls:
            call()
        tree.check(), slots.check(), decode.check(), prefill.check()
        del graph
    tt.agree(b.run(), b.want(), "f32")
    hip.synchronize()
    b.cache.set_stream(None)


def test_a_capture_that_forks_and_joins(device, oracle):
    """Captured from the cache's stream, launches on another one join the capture and
    come back to it."""
    tt.say("tree captured, two streams")
    b = tt.Batch(device, oracle, 4, 2, 64, [400, 30], [tt.chain(3), [-1]], seed=2)
    own, other = hip.Stream(), hip.Stream()
    hip.synchronize()
    b.cache.set_stream(own.h)
    with tt.hip_rows(b) as d:
        plan = attention.TreePlan(b.cache, b.seqs, b.nodes, b.parents, 4, 1 << 20)
        graph = tt.Graph(own.h, lambda: plan.launch(0, d.q.ptr, d.k.ptr, d.v.ptr, d.out.ptr, stream=other.h))
        for _ in range(3):
            d.out.zero()
            hip.synchronize()
            graph.replay()
            tt.agree(d.out.numpy()[: b.rows], b.want(), "f32")
            tt.agree(b.run(), b.want(), "f32")
        del graph
    hip.synchronize()
    b.cache.set_stream(None)
