"""Into how many parts packed sequences' dK and dV are split, as the size of the workspace shows."""

import ctypes

import pytest

from gefen_amd import _lib
from test_cpu_layer_ops import FAKE, attention_task


def partial_floats(sequences, each, heads, kv_heads, width, dtype=_lib.BF16):
    """Floats of the workspace behind the row statistics."""
    tokens = sequences * each
    t = attention_task(batch=1, queries=tokens, keys=tokens, heads=heads, kv_heads=kv_heads, width=width, offsets=FAKE,
                       sequences=sequences, dtype=dtype)
    n = int(_lib.load().gefen_attention_backward_workspace_size(ctypes.byref(t)))
    assert n > 0
    return n / 4 - tokens * heads


@pytest.mark.parametrize("sequences,each,heads,kv_heads,width", [(64, 128, 8, 8, 128), (256, 64, 32, 8, 64),
                                                                 (32, 192, 16, 16, 64), (1000, 7, 32, 32, 128)])
def test_short_sequences_are_not_split_for_their_lengths(sequences, each, heads, kv_heads, width):
    """A part would have less than four tiles of a sequence, and float32 copies of dK and dV to write."""
    assert partial_floats(sequences, each, heads, kv_heads, width) < 64


def test_long_sequences_are():
    """Four parts of dK and of dV."""
    for sequences, each in ((11, 1490), (4, 4096), (16, 512)):
        size = sequences * each * 8 * 64
        assert abs(partial_floats(sequences, each, 32, 8, 64) - 4 * 2 * size) < 64
