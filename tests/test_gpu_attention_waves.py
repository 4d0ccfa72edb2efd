"""attention of heads of up to 64 with more workgroups than two, and than three, a compute unit, against
its definition in float64 (bounds: test_gpu_attention)."""

import math

import pytest
import torch

from test_gpu_attention import NAMES, call, definition, make, visible, within

pytestmark = pytest.mark.gpu


def off_alignment(t):
    """A copy one element off any alignment."""
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
    return buf.copy_(t)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d,aligned", [(63, True), (64, False), (33, True), (31, True)])
@pytest.mark.parametrize("b", [15, 30])
def test_rows_that_come_through_registers(dtype, d, aligned, b):
    q, k, v, go = make(dtype, b, 500, 300, 10, 5, d)  # 8 x 5 x b workgroups of queries
    lengths = [(37 * i) % 301 for i in range(b)]
    if not aligned:
        q, k, v, go = (off_alignment(t) for t in (q, k, v, go))
    for i, n in enumerate(lengths):
        k[i, n:], v[i, n:] = math.nan, math.inf
    got = call(q, k, v, go, causal=True, key_lengths=torch.tensor(lengths, device="cuda"))
    for i, n in enumerate(lengths):
        k[i, n:], v[i, n:] = 0.0, 0.0
    want, bounds = definition(q, k, v, go, visible(b, 500, 300, True, lengths), dtype)
    for x, w, e, name in zip(got, want, bounds, NAMES):
        within(x, w, e, name)
