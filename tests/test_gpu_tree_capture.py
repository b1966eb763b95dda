"""Captured launches of tree and slot plans: what a graph may and may not hold."""

import numpy as np
import pytest

import test_gpu_tree as tt
from tvara_amd import attention, hip
from tvara_amd.kv import SlotPlan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("what", ["attention", "write"])
def test_replays_leave_blocks_handed_out_before(device, oracle, what):
    """A block that still waits for its zeros when a plan is made: a graph of the plan's
    launches does not clear it, however often it is replayed."""
    tt.say("tree captured, block handed out", what)
    b = tt.Batch(device, oracle, 4, 2, 64, [40], [tt.chain(3)], seed=2, spare=2)
    stream = hip.Stream()
    b.cache.set_stream(stream.h)
    h = b.cache.allocate()
    up = hip.DeviceArray.from_numpy
    with tt.hip_rows(b) as d:
        if what == "attention":
            plan = attention.TreePlan(b.cache, b.seqs, b.nodes, b.parents, 4, 1 << 20)
            launch = lambda: plan.launch(0, d.q.ptr, d.k.ptr, d.v.ptr, d.out.ptr, stream=stream.h)  # noqa: E731
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
    b.cache.set_stream(None)
