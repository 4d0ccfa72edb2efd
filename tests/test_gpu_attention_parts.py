"""Packed sequences whose dK and dV take a part, two and four, against the definition in float64
(bounds: test_gpu_attention)."""

import pytest
import torch

from test_gpu_attention import NAMES, call, definition, make, visible, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lengths,heads,kv_heads", [([100] * 20 + [0, 1] + [95] * 20, 32, 8), ([60] * 33, 16, 16),
                                                    ([1500, 1, 700], 16, 8)])
def test_packed_sequences_of_all_lengths(dtype, lengths, heads, kv_heads):
    n, d = sum(lengths), 40
    offsets = torch.tensor([0] + lengths).cumsum(0)
    q, k, v, go = make(dtype, 1, n, n, heads, kv_heads, d)
    got = call(q[0], k[0], v[0], go[0], causal=True, offsets=offsets.cuda())
    want, bounds = definition(q, k, v, go, visible(1, n, n, True, offsets=offsets.tolist()), dtype)
    for x, w, e, name in zip(got, want, bounds, NAMES):
        within(x[None], w, e, name)
