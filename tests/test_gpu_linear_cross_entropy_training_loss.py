"""The loss of a call that keeps values for its gradients is the loss of one that does not.

Both are the same sums: they may differ by the order of a few float32 operations, two units in
the last place of the loss."""

import pytest
import torch

from test_gpu_linear_cross_entropy import F, lce, make

pytestmark = pytest.mark.gpu


def same(a, b):
    return bool(((a - b).abs() <= 4 * F * b.abs()).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,v", [(40, 5000), (100, 5000), (300, 40000)])
def test_coherent_columns(dtype, n, v):
    """Columns of equal logits a little below the one that leads each slot of 64: an error of
    exp is the same in all of them."""
    h = torch.zeros(n, 64, device="cuda")
    h[:, 0] = torch.linspace(0.25, 3.0, n, device="cuda")
    w = torch.zeros(v, 64, device="cuda")
    w[::64, 0] = 1.0
    y = torch.arange(n, device="cuda")
    t = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[dtype]
    h, w = h.to(t), w.to(t)
    a = h[:, 0].double()
    lead, rest = (v + 63) // 64, v - (v + 63) // 64
    want = (lead * a.exp() + rest).log() - a * (y % 64 == 0)
    plain = lce(h, w, y, reduction="none")
    hg, wg = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    assert same(lce(hg, wg, y, reduction="none").detach(), plain)
    assert same(lce(hg, wg, y).detach(), lce(h, w, y))
    # exp to a few roundings at arguments up to 3, sums of up to 64 and v / 64 terms in float32
    assert bool(((plain.double() - want).abs() <= (8 + 64) * F + 2 * F * want).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_any_logits(dtype):
    h, w, y = make(300, 4000, 192, dtype, seed=60, ignored=0.2)
    hg, wg = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    assert same(lce(hg, wg, y, reduction="none").detach(), lce(h, w, y, reduction="none"))
    assert same(lce(hg, wg, y, reduction="sum").detach(), lce(h, w, y, reduction="sum"))
