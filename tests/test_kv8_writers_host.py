"""What the writers of an 8-bit cache refuse beside their sizes, without a GPU: caches whose rows or scales overlap."""

import pytest

from akv_amd import _lib
from tests.test_kv8_host import APPEND, MOVE, READ, _call


@pytest.mark.parametrize("name", [APPEND, MOVE])
@pytest.mark.parametrize("change", [
    dict(ks_stride_block=0), dict(vs_stride_block=0), dict(ks_stride_head=0), dict(vs_stride_head=0),
    dict(k_stride_slot=0), dict(v_stride_slot=32), dict(k_stride_head=63), dict(v_stride_head=-63),
    dict(scale_block=8, ks_stride_block=0), dict(ks_stride_block=0, ks_stride_head=0),
])
def test_writers_refuse_rows_and_scales_that_overlap(name, change):
    assert _call(name, **change) == _lib.AKV_EINVAL
    assert "overlap" in _lib.last_error()


@pytest.mark.parametrize("name", [APPEND, MOVE])
def test_strides_of_one_say_nothing(name):
    """Of one head, slot or block; refused for what else is wrong with these calls."""
    heads = "kv_heads" if name == APPEND else "n_heads"
    too_large = dict(n_tokens=(1 << 31) - 1)
    for change in (dict(scale_block=16, ks_stride_block=0, vs_stride_block=0),
                   {heads: 1, "k_stride_head": 0, "v_stride_head": 0, "ks_stride_head": 0, "vs_stride_head": 0},
                   dict(pool_slots=1, k_stride_slot=0, v_stride_slot=0, ks_stride_block=0, vs_stride_block=0)):
        assert _call(name, **change, **too_large) == _lib.AKV_EINVAL
        assert "batch too large" in _lib.last_error()


def test_a_pool_of_nothing_has_no_strides():
    strides = {name: 0 for name in ("k_stride_slot", "k_stride_head", "v_stride_slot", "v_stride_head", "ks_stride_block",
                                    "ks_stride_head", "vs_stride_block", "vs_stride_head")}
    pool = dict(k_pool=None, v_pool=None, k_scales=None, v_scales=None)
    assert _call(APPEND, pool_slots=0, q_heads=0, **pool, **strides) == 0
    assert _call(MOVE, pool_slots=0, **strides) == 0


def test_scales_of_a_layer_can_be_read():
    """One scale for all blocks and heads is no reason to refuse the attention."""
    assert _call(READ, ks_stride_block=0, ks_stride_head=0, vs_stride_block=0, vs_stride_head=0, workspace_bytes=0) \
        == _lib.AKV_EINVAL
    assert "workspace" in _lib.last_error()
