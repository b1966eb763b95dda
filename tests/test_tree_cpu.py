"""Entry points of speculative decoding with trees refuse closed handles (no
device calls: CPU only)."""

import numpy as np
import pytest

from tvara_amd import _capi, attention


def test_closed_handles_are_refused():
    lib = _capi.lib()
    n = np.zeros(1, np.uint64)
    for rc in (lib.tvara_kv_reserve(None, None, 0, None), lib.tvara_kv_pool_address(None, None, None),
               lib.tvara_tree_plan_launch(None, 0, None, None, None, 0, None, None),
               lib.tvara_tree_plan_accept(None, None, None, None, 1, 0, None, 0, None, None, None),
               lib.tvara_tree_plan_check(None),
               lib.tvara_attn_tree(None, None, 0, 0, 1, 1, None, None, None, None, None, None, None, 0, 0),
               lib.tvara_slot_plan_build(None, None, None, 0, 0, None, None, None, None, 0, None),
               lib.tvara_slot_plan_write(None, None, None, 0, None, None, 0, 0, 0, None),
               lib.tvara_slot_plan_check(None)):
        assert rc == _capi.INVALID
    assert not lib.tvara_tree_plan_create(None, None, 0, 1, 1, None, None, None, 0)
    assert lib.tvara_last_status() == _capi.INVALID
    assert not lib.tvara_slot_plan_create(None, None, 0)
    lib.tvara_tree_plan_destroy(None)
    lib.tvara_slot_plan_destroy(None)
    assert n[0] == 0


def test_closed_model_is_refused():
    lib = _capi.lib()
    assert lib.tvara_sequences_verify_trees(None, None, 0, None, None, None, None, None, None, None) == -1
    assert lib.tvara_last_error() == b"invalid batch buffers"


def test_trees_of_unequal_lists_are_refused():
    for nodes, parents in (([1], [-1, 0]), ([1, 2], [-1, -1]), ([], [])):
        with pytest.raises(_capi.InvalidArgument):
            attention._trees([1, 2], nodes, parents, None)


@pytest.mark.parametrize("parents,visible", [([-1, 2**32 - 1], None), (np.array([-1, 2**32]), None), ([-1, 0.5], None),
                                             ([-1, 0], -1), ([-1, 0], np.array([-1])), ([-1, 0], np.array([3.5]))])
def test_numbers_that_would_change_are_refused(parents, visible):
    """A parent of 2^32 - 1 is no -1, a visible length of -1 not all of the sequence."""
    with pytest.raises(_capi.InvalidArgument):
        attention._trees([1], [2], parents, visible)


def test_whole_numbers_of_any_type_are_taken():
    for dtype in (np.int64, np.int32, np.int8, np.float64):
        (seqs, nodes, parents, visible), _ = attention._trees([1, 2], np.array([2, 0], dtype), np.array([-1, 0], dtype), [7, 0])
        assert nodes.tolist() == [2, 0] and parents.tolist() == [-1, 0] and visible.tolist() == [7, 0]
    (_, nodes, parents, _), _ = attention._trees([1], [0], [], None)
    assert nodes.tolist() == [0] and parents.size == 0
