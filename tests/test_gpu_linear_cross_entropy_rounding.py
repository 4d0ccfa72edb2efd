"""Gradients of 16-bit operands are rounded to their type once, whatever the gradient of the
loss is."""

import pytest
import torch

from test_gpu_linear_cross_entropy import IGNORE, U, definition, lce, make

pytestmark = pytest.mark.gpu
THIRD = 1.0 / 3.0


def gradients(h, w, y, scale, **k):
    h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    return torch.autograd.grad(lce(h, w, y, **k) * scale, (h, w))


def half_spacing(x, dtype):
    """Half the distance between two numbers of the dtype at x."""
    bits = 8 if dtype == "bf16" else 11
    return torch.ldexp(torch.ones_like(x), torch.frexp(x).exponent - bits - 1)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_every_element_is_rounded_once(dtype, reduction):
    """Up to 64 rows G has twice the type's bits: 2^-14 covers them and the logits' errors
    ((d + 2) 2^-24 of at most 40 at a width of 16), so what remains is one rounding."""
    h, w, y = make(48, 500, 16, dtype, seed=70, ignored=0.1)
    got = gradients(h, w, y, THIRD, reduction=reduction)
    third = float(torch.tensor(1.0) * THIRD)
    count = int((y != IGNORE).sum())
    c = torch.full((48,), third / (count if reduction == "mean" else 1), device="cuda", dtype=torch.float64)
    ref = definition(h, w, y, dtype, row_grad=c)
    logits = torch.mm(h.double(), w.double().t())
    p = torch.softmax(logits, 1)
    q = torch.zeros_like(p).scatter_(1, y.clamp(min=0)[:, None], 1.0)
    g = ((p - q).abs() + p) * torch.where(y != IGNORE, c, torch.zeros_like(c))[:, None]
    size = torch.mm(g, w.double().abs()), torch.mm(g.t().contiguous(), h.double().abs())
    floor = 2.0 ** -25 if dtype == "f16" else 0.0
    for x, want, s in zip(got, (ref[2], ref[4]), size):
        bound = half_spacing(want, dtype) + 2.0 ** -14 * s + floor
        worst = float(((x.double() - want).abs() / bound.clamp(min=1e-300)).max())
        assert worst <= 1.0, worst


@pytest.mark.parametrize("n,limit", [(400, None), (900, 4 << 20)])
def test_a_loss_gradient_adds_no_error(n, limit):
    """Positions that fit the workspace together and ones taken in pieces: the error of a
    third of the loss is that of the loss, to within a twentieth (a second rounding adds a
    fifth)."""
    h, w, y = make(n, 4000, 96, "bf16", seed=71)
    ref = definition(h, w, y, "bf16")
    one = gradients(h, w, y, 1.0, workspace_limit=limit)
    third = gradients(h, w, y, THIRD, workspace_limit=limit)
    for a, b, want in zip(one, third, (ref[2], ref[4])):
        plain = float((a.double() - want).norm() / want.norm())
        scaled = float((b.double() - THIRD * want).norm() / (THIRD * want.norm()))
        assert plain < U["bf16"]
        assert scaled <= 1.05 * plain, (plain, scaled)
