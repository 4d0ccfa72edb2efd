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


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 40, 24])
@pytest.mark.parametrize("b", [12, 15, 30])
def test_few_and_many_workgroups(dtype, d, b):
    """480, 600 and 1200 of queries: two waves a SIMD, and three."""
    q, k, v, go = make(dtype, b, 500, 300, 10, 5, d)
    lengths = [(37 * i) % 301 for i in range(b)]
    for i, n in enumerate(lengths):
        k[i, n:], v[i, n:] = math.nan, math.inf
    got = call(q, k, v, go, causal=True, key_lengths=torch.tensor(lengths, device="cuda"))
    for i, n in enumerate(lengths):
        k[i, n:], v[i, n:] = 0.0, 0.0
    want, bounds = definition(q, k, v, go, visible(b, 500, 300, True, lengths), dtype)
    for x, w, e, name in zip(got, want, bounds, NAMES):
        within(x, w, e, name)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 33])
def test_packed_sequences_of_many_workgroups(dtype, d):
    q, k, v, go = make(dtype, 1, 2000, 2000, 48, 48, d)  # 16 x 48
    offsets = [3, 4, 300, 300, 1111, 1990]
    got = call(q[0], k[0], v[0], go[0], causal=True, offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"))
    want, bounds = definition(q, k, v, go, visible(1, 2000, 2000, True, offsets=offsets), dtype)
    for x, w, e, name in zip(got, want, bounds, NAMES):
        within(x[None], w, e, name)


def test_a_call_of_few_workgroups_gives_the_rows_of_one_of_many():
    q, k, v, go = make("bf16", 30, 500, 300, 10, 5, 64)
    many = call(q, k, v, go, causal=True)
    few = call(*(t[:12] for t in (q, k, v, go)), causal=True)
    assert all(torch.equal(x[:12], y) for x, y in zip(many, few))
