"""float32 hidden states whose rows differ widely in size: a row's loss and its gradient do not
depend on the others.

Bounds: test_gpu_linear_cross_entropy.py.  The rows of a large size have logits beyond any
loss; what they may change is dW, to which they add far larger terms than the others do."""

import pytest
import torch

from test_gpu_linear_cross_entropy import IGNORE, definition, lce, make, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [5, 40, 300, 1100])
@pytest.mark.parametrize("size", [1e9, 1e15, 1e30])
def test_a_row_of_a_large_size_leaves_the_others_alone(size, n):
    h, w, y = make(n, 700, 96, "f32", seed=80, ignored=0.1)
    y[2] = 3
    ref = definition(h, w, y, "f32", mean=False)
    big = h.clone()
    big[2] *= size
    rest = torch.arange(n, device="cuda") != 2
    rows = lce(big, w, y, reduction="none")
    within(rows[rest], ref[0][rest], ref[1][rest], "losses")
    for reduction in ("sum", "none"):
        g = big.clone().requires_grad_(True)
        lce(g, w, y, reduction=reduction).sum().backward()
        within(g.grad[rest], ref[2][rest], ref[3][rest], "dh")
        assert bool((g.grad[y == IGNORE] == 0).all())


def test_rows_of_every_size():
    """Sizes from 2^-60 to 2^60 and zero: the losses and gradients of hidden."""
    h, w, y = make(121, 500, 64, "f32", seed=81)
    h *= torch.ldexp(torch.ones(121, device="cuda"), torch.arange(121, device="cuda") - 60)[:, None]
    h[50] = 0.0
    ref = definition(h, w, y, "f32", mean=False)
    h.requires_grad_(True)
    rows = lce(h, w, y, reduction="none")
    rows.sum().backward()
    within(rows.detach(), ref[0], ref[1], "losses")
    within(h.grad, ref[2], ref[3], "dh")


@pytest.mark.parametrize("reduction", ["sum", "none"])
@pytest.mark.parametrize("low", [2.0 ** -20, 2.0 ** -27])
def test_weight_gradients_of_smaller_rows(low, reduction):
    """Rows down to 2^-27 of the largest reach dW with what float32 keeps of them, beside
    rows that do not reach the same columns."""
    n, v = 300, 640
    rows = torch.arange(n, device="cuda")
    small = rows % 2 == 1
    y = torch.where(small, 320 + rows % 300, rows % 300)
    h = torch.zeros(n, v, device="cuda")
    h[rows, y] = torch.where(small, 40.0 * low, 40.0)
    w = torch.eye(v, device="cuda")
    w[320:] /= low  # the logits of small rows are those of the others
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    loss = lce(h, w, y, reduction=reduction)
    loss.sum().backward()
    ref = definition(h.detach(), w.detach(), y, "f32", mean=False)
    # what a G of e^-40 keeps above its end at 2^-50
    end = 2.0 ** -50 * h.detach().double().abs().sum(0)
    within(w.grad, ref[4], ref[5] + end, "dw")
