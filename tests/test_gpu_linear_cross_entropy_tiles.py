"""linear_cross_entropy where its kernels change over: sizes on either side of a rule,
tiles that end inside the vocabulary, the rows or the width, K cut into parts; and the
scales that float32 operands may have.  Bounds: test_gpu_linear_cross_entropy.py."""

import math

import pytest
import torch

from test_gpu_linear_cross_entropy import F, IGNORE, definition, lce, make, within

pytestmark = pytest.mark.gpu


def both(h, w, y, dtype, floor=0.0, **k):
    h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = lce(h, w, y, **k)
    loss.backward()
    rows, erows, dh, edh, dw, edw = definition(h.detach(), w.detach(), y, dtype, k.get("label_smoothing", 0.0))
    count = int((y != IGNORE).sum())
    assert abs(float(loss.detach()) - float(rows.sum()) / count) <= float(erows.sum()) / count + 2 * F * abs(float(loss.detach()))
    within(h.grad, dh, edh + floor, "dh")
    within(w.grad, dw, edw + floor, "dw")


# rows: one and two planes of G (64 / 65), the narrow tile (32 / 33), rows selected by every
# workgroup or by one (1024 / 1025); columns on both sides of a slot, a tile, G's row length
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,v,d", [(32, 1000, 64), (33, 1000, 64), (64, 640, 130), (65, 640, 130), (1024, 300, 64),
                                   (1025, 300, 64), (100, 63, 64), (100, 64, 65), (100, 65, 63), (40, 255, 8),
                                   (40, 256, 9), (40, 257, 7)])
def test_on_either_side_of_a_rule(dtype, n, v, d):
    h, w, y = make(n, v, d, dtype, seed=30, ignored=0.1)
    y[0], y[n - 1] = v - 1, 0  # the last column of a partial slot, the first
    both(h, w, y, dtype)


# big tiles with edges, K of dh (the vocabulary) and of dW (the rows) cut into parts, most
# rows ignored so that the device finds fewer tiles than the host allowed for
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,v,d,ignored", [(700, 9000, 300, 0.0), (1100, 33000, 520, 0.3), (2500, 700, 260, 0.9),
                                           (300, 40000, 256, 0.5), (5000, 2100, 129, 0.0)])
def test_big_tiles_and_cut_products(dtype, n, v, d, ignored):
    h, w, y = make(n, v, d, dtype, seed=31, ignored=ignored)
    both(h, w, y, dtype, label_smoothing=0.1 if n == 700 else 0.0)


@pytest.mark.parametrize("live", [1, 2, 63, 64, 65, 255, 256, 257])
def test_few_rows_of_many_take_part(live):
    h, w, y = make(900, 3000, 96, "bf16", seed=32)
    keep = torch.randperm(900, generator=torch.Generator().manual_seed(live))[:live].cuda()
    z = torch.full_like(y, IGNORE)
    z[keep] = y[keep]
    both(h, w, z, "bf16")


@pytest.mark.parametrize("sh,sw", [(1e15, 1e-15), (1e-18, 1e18), (1e-3, 1e3)])
def test_float32_operands_of_any_scale(sh, sw):
    """The products bring each matrix to half precision's range by a power of two."""
    h, w, y = make(150, 900, 100, "f32", seed=33)
    both((h.double() * sh).float(), (w.double() * sw).float(), y, "f32")


def test_float32_elements_far_below_the_largest():
    """Rows of hidden and weight 2^-20 of the others keep their relative precision."""
    h, w, y = make(120, 640, 64, "f32", seed=34)
    h[::3] *= 2.0 ** -20
    w[::5] *= 2.0 ** -20
    both(h, w, y, "f32")


def test_smoothing_of_one_and_every_target_the_same():
    h, w, y = make(80, 333, 48, "bf16", seed=35)
    both(h, w, y, "bf16", label_smoothing=1.0)
    both(h, w, torch.full_like(y, 332), "bf16")


def test_single_rows_and_columns():
    """Widths of one leave probabilities far outside any range: what lies below the smallest
    one that is kept, times the other operand (below 2^16 here), is zero.  bfloat16 keeps
    down to 2^-126; the two half planes of a float32 G end at 2^-24 / (2^15 2^11)."""
    for n, v, d in [(1, 1, 1), (1, 1, 64), (3, 1, 7), (1, 5000, 1), (5000, 2, 3)]:
        for dtype in ("bf16", "f32"):
            h, w, y = make(n, v, d, dtype, seed=36)
            assert float(h.abs().max()) < 2.0 ** 16 and float(w.abs().max()) < 2.0 ** 16
            both(h, w, y, dtype, floor=2.0 ** -110 if dtype == "bf16" else 2.0 ** -34)


def test_more_rows_than_a_piece_holds_without_gradients():
    """Loss alone, positions in pieces of a small workspace."""
    h, w, y = make(3000, 4100, 64, "bf16", seed=37, ignored=0.2)
    got = lce(h, w, y, reduction="none", workspace_limit=1 << 20)
    rows, erows, *_ = definition(h, w, y, "bf16")
    within(got, rows, erows, "losses")
    assert torch.equal(got, lce(h, w, y, reduction="none"))


def test_workspace_is_bounded():
    """The memory of a training call stays by its limit, whatever the logits would take."""
    n, v, d = 20000, 30000, 64
    h, w, y = make(n, 100, d, "bf16", seed=38)
    w = torch.randn(v, d, device="cuda").bfloat16()
    h.requires_grad_(True)
    w.requires_grad_(True)
    limit = 64 << 20
    lce(h, w, y, workspace_limit=limit)  # warm
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    loss = lce(h, w, y, workspace_limit=limit)
    torch.cuda.synchronize()
    peak = torch.cuda.max_memory_allocated() - before
    grads = 2 * (n + v) * d
    # a copy of hidden, the float32 sum of dW, at most 256 MiB of partial tiles, 32 bytes a row
    assert peak <= limit + grads + 2 * (n + 512) * d + 4 * v * d + (256 << 20) + 64 * n + (1 << 20)
    assert peak < n * v * 2
    del loss


def test_gradient_of_the_loss_as_a_strided_or_narrow_tensor():
    h, w, y = make(50, 300, 64, "bf16", seed=39)
    h.requires_grad_(True)
    rows = lce(h, w, y, reduction="none")
    c = torch.randn(50, 2, device="cuda")
    a = torch.autograd.grad(rows, h, grad_outputs=c[:, 0], retain_graph=True)[0]
    b = torch.autograd.grad(rows, h, grad_outputs=c[:, 0].contiguous())[0]
    assert torch.equal(a, b)
    one = lce(h, w, y, reduction="none")
    one.sum().backward()  # an expanded gradient
    want = definition(h.detach(), w, y, "bf16", mean=False)
    within(h.grad, want[2], want[3], "dh of a sum")


def test_differentiating_twice_is_refused():
    h, w, y = make(20, 100, 32, "bf16", seed=40)
    h.requires_grad_(True)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(lce(h, w, y), h, create_graph=True)


def test_losses_of_a_batch_keep_its_shape():
    h, w, y = make(60, 100, 32, "bf16", seed=41)
    rows = lce(h.view(3, 4, 5, 32), w, y.view(3, 4, 5), reduction="none")
    assert rows.shape == (3, 4, 5) and rows.dtype == torch.float32
    assert not rows.requires_grad
    assert math.isclose(float(rows.double().mean()), float(lce(h, w, y)), rel_tol=1e-6)


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,v,d,ignored", [(1, 70, 9, 0.0), (60, 900, 64, 0.3), (300, 4100, 200, 0.0),
                                           (1100, 700, 130, 0.5), (40, 300, 16, 1.0)])
def test_gradients_of_kept_values_are_those_of_a_second_product(n, v, d, ignored, dtype, reduction):
    """The first backward starts from what the forward call kept, the second one of a retained
    graph from the operands, and a call in pieces keeps nothing."""
    h, w, y = make(n, v, d, dtype, seed=n, ignored=ignored)
    h.requires_grad_(True)
    w.requires_grad_(True)
    rows = lce(h, w, y, reduction=reduction, label_smoothing=0.1)
    c = torch.rand(rows.shape, generator=torch.Generator().manual_seed(2)).cuda() + 0.5
    if reduction == "mean":
        c = torch.ones_like(c)
    kept = torch.autograd.grad(rows, (h, w), grad_outputs=c, retain_graph=True)
    again = torch.autograd.grad(rows, (h, w), grad_outputs=c)
    assert torch.equal(kept[0], again[0]) and torch.equal(kept[1], again[1])
    assert not kept[0][y == -100].any()
    for i, x in enumerate((h, w)):
        alone = lce(h if i == 0 else h.detach(), w if i == 1 else w.detach(), y, reduction=reduction,
                    label_smoothing=0.1)
        assert torch.equal(alone, rows) or ignored == 1.0
        assert torch.equal(torch.autograd.grad(alone, x, grad_outputs=c)[0], kept[i])


def test_kept_values_outlive_other_calls_and_refuse_changed_operands():
    h, w, y = make(200, 3000, 96, "f16", seed=4)
    h.requires_grad_(True)
    w.requires_grad_(True)
    want = torch.autograd.grad(lce(h, w, y), (h, w))
    first = lce(h, w, y)
    second = lce(h * 2, w, y.flip(0))
    torch.autograd.grad(second, w)
    got = torch.autograd.grad(first, (h, w))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    loss = lce(h, w, y)
    with torch.no_grad():
        w.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_values_are_kept_only_within_the_limit():
    h, w, y = make(1000, 4096, 64, "f16", seed=6)
    h.requires_grad_(True)
    w.requires_grad_(True)
    lce(h, w, y).backward()  # the allocator's first blocks
    g = h.grad.clone(), w.grad.clone()

    def held(limit):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        loss = lce(h, w, y, workspace_limit=limit)
        after = torch.cuda.memory_allocated()
        got = torch.autograd.grad(loss, (h, w))
        return after - before, got

    much, a = held(None)
    little, b = held(1 << 20)
    assert much >= 1000 * 4096 * 2 and little <= 4096
    for x, z, r in zip(a, b, g):
        assert torch.equal(x, r)
        assert torch.allclose(z.float(), r.float(), rtol=2.0 ** -9, atol=2.0 ** -22)
