"""No-GPU checks of the draft-tree entry points: refusals that need no device, and what the binding refuses before it calls."""
import numpy as np
import pytest
from pooled_amd import capi


def test_no_context():
    L = capi.load()
    assert L.pa_set_rope_axes(None, 1, None) == capi.PA_ERR_INVALID
    assert L.pa_glue_kv_at(None, 0, None, 0, None, 0, None, 0, None, None, None, 0, 0, 1) == capi.PA_ERR_INVALID
    assert L.pa_attn_tree(None, 0, None, 0, None, 0, None, 1, 0, 1, None, 0, 0) == capi.PA_ERR_INVALID
    assert L.pa_kv_compact(None, 0, None, 1) == capi.PA_ERR_INVALID


def test_a_parent_comes_before_its_child():
    for parents in ([0], [-1, 2], [-1, 0, -2], [1, -1]):
        with pytest.raises(ValueError):
            capi.tree_of_parents(parents)
    assert np.array_equal(capi.tree_of_parents([-1, 0, -1, 2]), np.array([[1, 0, 0, 0], [1, 1, 0, 0], [0, 0, 1, 0], [0, 0, 1, 1]], bool))


def test_axes_are_refused_before_the_call():
    class Stub:
        cfg = dict(n_rot=8)
    for axes in ([0, 1, 2], [0, 1, 2, 4], [0, -1, 0, 0]):
        with pytest.raises(ValueError):
            capi.PooledAttn.set_rope_axes(Stub(), axes)
