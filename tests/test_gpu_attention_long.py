"""attention whose workgroups take several hundred tiles each, so that loads to LDS follow each
other for long, against its definition in float64 (bounds: test_gpu_attention)."""

import pytest
import torch

from test_gpu_attention import NAMES, call, definition, make, visible, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,d", [("f32", 128), ("f32", 100), ("f32", 64), ("bf16", 128), ("f16", 128), ("bf16", 64)])
def test_several_hundred_tiles_a_workgroup(dtype, d):
    """128 workgroups of queries (more than are split) over 313 tiles of keys, and 157 workgroups
    of keys over 4 x 64 tiles of queries."""
    b, sq, sk, h, hk = 1, 4096, 20000, 4, 1
    q, k, v, go = make(dtype, b, sq, sk, h, hk, d)
    got = call(q, k, v, go, causal=True)
    again = call(q, k, v, go, causal=True)
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    want, bounds = definition(q, k, v, go, visible(b, sq, sk, True), dtype)
    for x, w, e, name in zip(got, want, bounds, NAMES):
        within(x, w, e, name)
