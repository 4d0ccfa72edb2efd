"""Sizes that attention takes: those that all of its launches hold, in both directions."""

import ctypes

import pytest

from gefen_amd import _lib
from test_cpu_layer_ops import FAKE, attention_task

MOST = (1 << 24) - 1  # workgroups of 256 along one axis: fewer than 2^32 work items


def taken(**k):
    """Whether the sizes are in range: a backward workspace has some bytes for every valid task."""
    return int(_lib.load().gefen_attention_backward_workspace_size(ctypes.byref(attention_task(**k)))) > 0


@pytest.mark.parametrize("dtype", [_lib.F32, _lib.F16, _lib.BF16])
@pytest.mark.parametrize("kv_heads,heads", [(1, 1), (2, 8), (8, 8)])
def test_sizes_stop_where_a_launch_does(dtype, kv_heads, heads):
    def one(**k):
        return taken(dtype=dtype, kv_heads=kv_heads, heads=heads, width=8, **k)

    batch, group = MOST // kv_heads, heads // kv_heads
    for rows in ((1, 1), (0, 1), (1, 0), (128 // group, 128)):  # a block of each
        assert one(batch=batch, queries=rows[0], keys=rows[1])
        assert not one(batch=batch + 1, queries=rows[0], keys=rows[1])
    # two blocks of either
    assert one(batch=batch // 2, queries=1, keys=129)
    assert not one(batch=batch // 2 + 1, queries=1, keys=129)
    assert one(batch=batch // 2, queries=128 // group + 1, keys=1)
    assert not one(batch=batch // 2 + 1, queries=128 // group + 1, keys=1)


def test_what_is_too_large_is_refused_in_both_directions():
    lib = _lib.load()
    for k in (dict(batch=1 << 20, heads=16, kv_heads=16, queries=1, keys=1), dict(batch=1 << 19, queries=1, keys=2000)):
        t = attention_task(**k)
        assert lib.gefen_attention_forward(ctypes.byref(t), FAKE, 1 << 60, None) == _lib.GEFEN_EINVAL
        assert b"2^24" in lib.gefen_last_error()
        assert lib.gefen_attention_backward(ctypes.byref(t), FAKE, 1 << 60, None) == _lib.GEFEN_EINVAL
        assert b"2^24" in lib.gefen_last_error()
