"""Losses that are not reduced, whose gradients differ widely or are not finite.

Bounds: test_gpu_linear_cross_entropy.py; a row's gradients are off in proportion to its own
loss's gradient, whatever the others' are, and probabilities end where G or the values kept
for it do (END)."""

import math

import pytest
import torch

from test_gpu_linear_cross_entropy import IGNORE, definition, lce, make, within

pytestmark = pytest.mark.gpu

END = {"bf16": 2.0 ** -73, "f16": 2.0 ** -39, "f32": 2.0 ** -50}


def backward(h, w, y, c, **k):
    h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    rows = lce(h, w, y, reduction="none", **k)
    return torch.autograd.grad(rows, (h, w), grad_outputs=c)


# the ratio of half precision is what its output type can hold: rows of 2^11 and of 2^-19,
# and weights of about six
@pytest.mark.parametrize("n", [40, 100, 700])
@pytest.mark.parametrize("dtype,most,ratio", [("bf16", 1.0, 1e-14), ("f32", 1.0, 1e-6), ("f32", 1e3, 1e-12),
                                              ("f32", 1.0, 1e-14), ("f32", 1e-20, 1e-14), ("f16", 2.0 ** 11, 2.0 ** -30)])
def test_hidden_gradients_of_uneven_rows(dtype, most, ratio, n):
    h, w, y = make(n, 900, 128, dtype, seed=50, ignored=0.2)
    k = 32 if dtype == "f16" else 64
    h, w = h / k, w * k
    c = torch.full((n,), most, device="cuda")
    c[1::3] *= ratio
    c[2::9] *= -math.sqrt(ratio)
    dh, _ = backward(h, w, y, c)
    ref = definition(h, w, y, dtype, row_grad=c)
    within(dh, ref[2], ref[3], "dh")
    assert bool((dh[y == IGNORE] == 0).all())


@pytest.mark.parametrize("limit", [None, 1 << 20])
@pytest.mark.parametrize("dtype,most,ratio", [("bf16", 1.0, 1e-14), ("f32", 1.0, 1e-9), ("f32", 1.0, 1e-14),
                                              ("f16", 2.0 ** 8, 2.0 ** -22)])
def test_weight_gradients_of_uneven_rows(dtype, most, ratio, limit):
    """Rows of a small gradient, the only ones that reach their columns of an identity."""
    n, v = 700, 1024
    rows = torch.arange(n, device="cuda")
    small = rows % 2 == 1
    y = torch.where(small, 512 + rows % 512, rows % 500)
    h = torch.zeros(n, v, device="cuda")
    h[rows, y] = 60.0
    h[rows, torch.where(small, 512 + (rows + 7) % 512, (rows + 7) % 500)] = 59.0
    w = torch.eye(v, device="cuda")
    h, w = (h.half(), w.half()) if dtype == "f16" else (h.bfloat16(), w.bfloat16()) if dtype == "bf16" else (h, w)
    c = torch.where(small, torch.tensor(most * ratio, device="cuda"), torch.tensor(most, device="cuda"))
    dh, dw = backward(h, w, y, c, workspace_limit=limit)
    ref = definition(h, w, y, dtype, row_grad=c)
    assert float(ref[4][513:].abs().max(1).values.min()) > 0
    c = c.double().abs()[:, None]
    within(dh, ref[2], ref[3] + END[dtype] * c * w.double().abs().sum(0), "dh")
    # what 1e-14 of the largest keeps of a float32 gradient: half an ulp of the eleven bits above
    # the end of hidden's planes
    end = END[dtype] * (c * h.double().abs()).sum(0)
    within(dw, ref[4], ref[5] + end + (2.0 ** -11 * ref[4].abs() if ratio < 1e-12 else 0.0), "dw")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [40, 300])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_row_gradient_that_is_not_finite_stays_in_its_row(bad, n, dtype):
    h, w, y = make(n, 700, 96, dtype, seed=51, ignored=0.1)
    y[5] = 3
    g = torch.Generator().manual_seed(1)
    c = torch.randn(n, generator=g).cuda()
    ref = definition(h, w, y, dtype, row_grad=c)
    c[5] = bad
    dh, dw = backward(h, w, y, c)
    rest = torch.arange(n, device="cuda") != 5
    floor = 2.0 ** -39 * 4 * w.double().abs().sum(0) if dtype == "f16" else 0.0
    within(dh[rest], ref[2][rest], (ref[3] + floor)[rest], "dh of the other rows")
    assert not bool(torch.isfinite(dh[5]).any())
    assert not bool(torch.isfinite(dw).any())  # every column's gradient has that row in its sum


def test_only_row_gradients_that_are_not_finite_or_zero():
    h, w, y = make(80, 300, 64, "bf16", seed=52)
    c = torch.zeros(80, device="cuda")
    dh, dw = backward(h, w, y, c)
    assert bool((dh == 0).all()) and bool((dw == 0).all())
    c[7] = float("inf")
    dh, dw = backward(h, w, y, c)
    rest = torch.arange(80, device="cuda") != 7
    assert bool((dh[rest] == 0).all()) and not bool(torch.isfinite(dh[7]).any())
    assert not bool(torch.isfinite(dw).any())
