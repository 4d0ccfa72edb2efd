"""float16 gradients of rows that are almost certain: a competitor 12 to 22 nats below its
target, in the target's slot of 64 columns and outside of it.

Bounds: test_gpu_linear_cross_entropy.py.  With an identity as the weight every entry of dh
is one entry of G, so its relative error is seen."""

import pytest
import torch

from test_gpu_linear_cross_entropy import definition, lce, within

pytestmark = pytest.mark.gpu

TOP = 60.0  # the target's logit: columns at 0 are e^-60 of it


@pytest.mark.parametrize("n", [80, 300])
@pytest.mark.parametrize("gap", [12.0, 14.0, 16.0, 19.0, 22.0])
@pytest.mark.parametrize("v,away", [(64, 1), (192, 64)])
def test_a_competitor_far_below_the_target(v, away, gap, n):
    y = torch.arange(n, device="cuda") % v
    other = (y + away) % v
    rows = torch.arange(n, device="cuda")
    h = torch.zeros(n, v, device="cuda")
    h[rows, y] = TOP
    h[rows, other] = TOP - gap
    h, w = h.half().requires_grad_(True), torch.eye(v, device="cuda").half().requires_grad_(True)
    scale = torch.tensor(2.0 ** 20, device="cuda")  # 22 nats below one: 3e-10, in half's normal range
    lce(h, w, y, reduction="sum").backward(scale)
    _, _, dh, edh, dw, edw = definition(h.detach(), w.detach(), y, "f16", row_grad=scale.expand(n))
    assert float(dh[rows, other].min()) > 2.0 ** -14
    within(h.grad, dh, edh, "dh")
    within(w.grad, dw, edw, "dw")
