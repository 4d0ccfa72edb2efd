"""linear_cross_entropy against its definition in float64, and what it refuses.

Error bounds, element by element (u: half the spacing of the operands' dtype at 1, 2^-8
for bf16, 2^-11 for f16, 2^-24 for f32; f = 2^-24):

* a logit is a float32 sum of D exact products: off by at most (D + 2) f sum |h W|
  (float32 operands: six plane products, 6 D terms, and three parts below 2^-24 dropped);
* lse is off by the largest logit's error and a few float32 roundings; exp's own error
  (f times its argument) weighs with the probabilities, hence 16 f (1 + log V);
* G = exp(l - m) rounded, times exp(m - lse), rounded: 2 u p, and p times the errors of
  l and lse; float16 loses what lies 2^-25 below 2^-15;
* a gradient is the sum of those errors times the other operand, a float32 sum of K terms
  and one rounding to the dtype."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
F = 2.0 ** -24
IGNORE = -100


def lce(*a, **k):
    from gefen_amd import linear_cross_entropy

    return linear_cross_entropy(*a, **k)


def make(n, v, d, dtype, seed=0, ignored=0.0, pull=6.0, scale=1.0):
    g = torch.Generator().manual_seed(1000 * seed + n + 7 * v + 13 * d)
    w = torch.randn(v, d, generator=g, dtype=torch.float64) * (scale * 2.0 / math.sqrt(d))
    y = torch.randint(0, v, (n,), generator=g)
    h = torch.randn(n, d, generator=g, dtype=torch.float64)
    r = w[y]
    h += r * (pull * torch.rand(n, 1, generator=g, dtype=torch.float64) / r.square().sum(1, keepdim=True))
    drop = torch.rand(n, generator=g) < ignored
    y = torch.where(drop, torch.full_like(y, IGNORE), y)
    return h.to(DT[dtype]).cuda(), w.to(DT[dtype]).cuda(), y.cuda()


def definition(h, w, y, dtype, smoothing=0.0, row_grad=None, mean=True):
    """Row losses, gradients for row gradients c (mean: 1 / count), and their bounds, float64."""
    h, w = h.double(), w.double()
    n, d = h.shape
    v = w.shape[0]
    u = U[dtype]
    live = y != IGNORE
    logits = torch.mm(h, w.t().contiguous())
    size = torch.mm(h.abs(), w.abs().t().contiguous())
    terms = 6 * d + 8 if dtype == "f32" else d + 2
    el = terms * F * size
    lse = torch.logsumexp(logits, 1)
    at = y.clamp(min=0)[:, None]
    ly = logits.gather(1, at)[:, 0]
    loss = (1 - smoothing) * (lse - ly) + smoothing * (lse - logits.mean(1))
    elmax = el.max(1).values
    eloss = 2 * elmax + 16 * F * (1 + math.log(v)) + 4 * F * (lse.abs() + ly.abs())
    if smoothing:
        eloss = eloss + (v + 4) * F * logits.abs().mean(1)
    zero = torch.zeros_like(loss)
    loss, eloss = torch.where(live, loss, zero), torch.where(live, eloss, zero)
    p = (logits - lse[:, None]).exp()
    q = torch.full_like(p, smoothing / v)
    q.scatter_add_(1, at, torch.full_like(ly, 1 - smoothing)[:, None])
    g = p - q
    drel = (el + elmax[:, None]) + 16 * F * (1 + math.log(v)) + 4 * F * (logits.abs() + lse.abs()[:, None])
    eg = p * (2.5 * u + 1.5 * drel) + (u + 2 * F) * g.abs() + 4 * F * (p + q)
    if dtype == "f16":
        eg = eg + 2.0 ** -39
    c = row_grad.double() if row_grad is not None else torch.full((n,), 1.0 / max(1, int(live.sum())) if mean else 1.0,
                                                                  dtype=torch.float64, device=h.device)
    c = torch.where(live, c, torch.zeros_like(c))[:, None]
    g, eg = g * c, eg * c.abs()
    k = 6.0 if dtype == "f32" else 1.0
    h0, w0 = h.abs(), w.abs()
    dh, dw = torch.mm(g, w), torch.mm(g.t().contiguous(), h)
    # a row weight is g / max|g|, applied and undone: two more roundings
    edh = torch.mm(eg, w0) + ((k * v + 16) * F) * torch.mm(g.abs(), w0) + (u + 4 * F) * dh.abs()
    edw = torch.mm(eg.t().contiguous(), h0) + ((k * n + 16) * F) * torch.mm(g.abs().t().contiguous(), h0) + (u + 4 * F) * dw.abs()
    if dtype == "f16":  # half's subnormal spacing
        edh, edw = edh + 2.0 ** -24, edw + 2.0 ** -24
    return loss, eloss, dh, edh, dw, edw


def within(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, what
    assert bool(torch.isfinite(got).all()), what
    bad = (got - want).abs() > bound
    assert not bool(bad.any()), "{}: {} of {} outside, worst {:.3g} of its bound".format(
        what, int(bad.sum()), bad.numel(), float(((got - want).abs() / bound.clamp(min=1e-300)).max()))


SIZES = [(1, 7, 1), (1, 300, 64), (2, 1, 5), (5, 1000, 96), (33, 257, 65), (64, 513, 128), (129, 1000, 200),
         (300, 4000, 192), (257, 129, 1001), (700, 260, 64), (31, 5003, 320), (1030, 8200, 72), (513, 16500, 256)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,v,d", SIZES)
def test_loss_and_gradients_match_the_definition(dtype, n, v, d):
    h, w, y = make(n, v, d, dtype, ignored=0.2 if n > 4 else 0.0)
    if not bool((y != IGNORE).any()):
        y[0] = 0
    h.requires_grad_(True)
    w.requires_grad_(True)
    loss = lce(h, w, y)
    assert loss.dtype == torch.float32 and loss.dim() == 0
    loss.backward()
    rows, erows, dh, edh, dw, edw = definition(h.detach(), w.detach(), y, dtype)
    count = int((y != IGNORE).sum())
    assert abs(float(loss) - float(rows.sum()) / count) <= float(erows.sum()) / count + 2 * F * abs(float(loss))
    within(h.grad, dh, edh, "dh")
    within(w.grad, dw, edw, "dw")
    with torch.no_grad():
        got = lce(h, w, y, reduction="none")
    within(got, rows, erows, "losses")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,v,d,limit", [(70, 777, 130, None), (1500, 900, 64, 1 << 20), (900, 5000, 100, 6 << 20)])
def test_smoothing_row_gradients_and_pieces(dtype, n, v, d, limit):
    """Per-row gradients (of either sign, some zero), label smoothing, and positions taken
    in pieces of a small workspace."""
    h, w, y = make(n, v, d, dtype, seed=1, ignored=0.3)
    h.requires_grad_(True)
    w.requires_grad_(True)
    c = torch.randn(n, device="cuda")
    c[::7] = 0.0
    rows = lce(h, w, y, reduction="none", label_smoothing=0.1, workspace_limit=limit)
    rows.backward(c)
    want, ewant, dh, edh, dw, edw = definition(h.detach(), w.detach(), y, dtype, 0.1, row_grad=c)
    within(rows.detach(), want, ewant, "losses")
    # rows of a small weight share the largest one's absolute floor in half precision
    if dtype == "f16":
        edw = edw + 2.0 ** -39 * float(c.abs().max()) * h.detach().double().abs().sum(0)
        edh = edh + 2.0 ** -39 * float(c.abs().max()) * w.detach().double().abs().sum(0)
    within(h.grad, dh, edh, "dh")
    within(w.grad, dw, edw, "dw")
    h.grad = w.grad = None
    loss = lce(h, w, y, reduction="sum", workspace_limit=limit)
    loss.backward()
    want, ewant, dh, edh, dw, edw = definition(h.detach(), w.detach(), y, dtype, mean=False)
    assert abs(float(loss) - float(want.sum())) <= float(ewant.sum()) + 2 * F * float(want.sum())
    within(h.grad, dh, edh, "dh sum")
    within(w.grad, dw, edw, "dw sum")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_any_strides(dtype):
    """A transposed weight, rows that start off any alignment, batched hidden states,
    int32 targets, one row broadcast."""
    h, w, y = make(60, 400, 128, dtype, seed=2, ignored=0.1)
    want = definition(h, w, y, dtype)
    wide = torch.zeros(400, 131, dtype=w.dtype, device="cuda")
    wide[:, 3:] = w
    big = torch.zeros(60, 2, 128, dtype=h.dtype, device="cuda")
    big[:, 1] = h
    forms = [(h, w.t().contiguous().t(), y), (h, wide[:, 3:], y), (big[:, 1], w, y.int()),
             (h.view(3, 20, 128), w, y.view(3, 20)), (h.t().contiguous().t(), w, y)]
    for hh, ww, yy in forms:
        hh, ww = hh.detach().requires_grad_(True), ww.detach().requires_grad_(True)
        lce(hh, ww, yy).backward()
        within(hh.grad.reshape(60, 128), want[2], want[3], "dh")
        within(ww.grad, want[4], want[5], "dw")
    one = h[:1].expand(60, 128)
    got = lce(one, w, y, reduction="none")
    ref = definition(one, w, y, dtype)
    within(got, ref[0], ref[1], "broadcast row")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_masked_positions_reach_nothing(dtype):
    h, w, y = make(200, 600, 96, dtype, seed=3, ignored=0.4)
    dead = y == IGNORE
    want = definition(h, w, y, dtype)
    h = h.clone()
    h[dead] = float("nan")
    h[torch.nonzero(dead)[0, 0]] = float("inf")
    h.requires_grad_(True)
    w.requires_grad_(True)
    lce(h, w, y).backward()
    assert bool((h.grad[dead] == 0).all())
    within(h.grad[~dead], want[2][~dead], want[3][~dead], "dh")
    within(w.grad, want[4], want[5], "dw")
    # another ignore_index, one that is a column's number too
    y2 = torch.where(dead, torch.full_like(y, 5), torch.where(y == 5, torch.full_like(y, 6), y))
    rows = lce(h.detach(), w.detach(), y2, ignore_index=5, reduction="none")
    assert bool((rows[dead] == 0).all()) and bool(torch.isfinite(rows).all())


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_no_position_and_none_that_counts(reduction):
    h, w, y = make(40, 300, 64, "bf16", seed=4)
    for hh, yy in ((h, torch.full_like(y, IGNORE)), (h[:0], y[:0])):
        hh, ww = hh.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = lce(hh, ww, yy, reduction=reduction)
        if reduction == "mean":
            assert bool(torch.isnan(loss))
        else:
            assert bool((loss == 0).all()) and loss.shape == (() if reduction == "sum" else yy.shape)
        loss.sum().backward()
        assert bool((hh.grad == 0).all()) and bool((ww.grad == 0).all())


def test_targets_outside_the_columns_are_not_a_number():
    h, w, y = make(40, 300, 64, "bf16", seed=5)
    want = definition(h, w, y, "bf16")
    y[3], y[11] = 300, -1
    rows = lce(h, w, y, reduction="none")
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[3] = bad[11] = True
    assert bool(torch.isnan(rows[bad]).all())
    within(rows[~bad], want[0][~bad], want[1][~bad], "other rows")
    assert bool(torch.isnan(lce(h, w, y)))


def test_non_finite_and_large_values():
    """Rows of NaN or infinite hidden states have NaN losses and leave the others alone;
    logits in the thousands neither overflow nor vanish; a column of -inf counts for
    nothing; one certain column leaves a loss and gradients of (nearly) nothing."""
    h, w, y = make(50, 700, 64, "f32", seed=6)
    want = definition(h, w, y, "f32")
    hb = h.clone()
    hb[4, 7], hb[9, 0] = float("nan"), float("inf")
    rows = lce(hb, w, y, reduction="none")
    bad = torch.zeros(50, dtype=torch.bool, device="cuda")
    bad[4] = bad[9] = True
    assert bool(torch.isnan(rows[bad]).all())
    within(rows[~bad], want[0][~bad], want[1][~bad], "other rows")
    big = lce(h * 1000, w, y, reduction="none")
    ref = definition(h * 1000, w, y, "f32")
    within(big, ref[0], ref[1], "large logits")
    ha = h.abs() + 0.5
    wn = w.clone()
    wn[13] = -float("inf")
    keep = torch.arange(700, device="cuda") != 13
    y2 = torch.where(y == 13, torch.zeros_like(y), y)
    rows = lce(ha, wn, y2, reduction="none")
    ref = definition(ha, wn[keep], torch.where(y2 > 13, y2 - 1, y2), "f32")
    within(rows, ref[0], ref[1], "a column of -inf")
    hc = (w[y] * 400).to(torch.bfloat16)
    wb = w.to(torch.bfloat16)
    hc.requires_grad_(True)
    loss = lce(hc, wb, y)
    loss.backward()
    assert float(loss) < 1e-6 and float(hc.grad.abs().max()) < 1e-6


def test_half_gradients_take_the_loss_scale_before_rounding():
    h, w, y = make(300, 2000, 64, "f16", seed=7)
    h.requires_grad_(True)
    w.requires_grad_(True)
    scale = 1024.0
    (lce(h, w, y) * scale).backward()
    _, _, dh, edh, dw, edw = definition(h.detach(), w.detach(), y, "f16")
    within(h.grad, dh * scale, (edh - 2.0 ** -24) * scale + 2.0 ** -24, "dh")
    within(w.grad, dw * scale, (edw - 2.0 ** -24) * scale + 2.0 ** -24, "dw")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_a_scaled_loss_a_second_backward_and_one_gradient_alone(dtype):
    h, w, y = make(100, 500, 72, dtype, seed=8)
    h.requires_grad_(True)
    w.requires_grad_(True)
    _, _, dh, edh, dw, edw = definition(h.detach(), w.detach(), y, dtype)
    loss = lce(h, w, y)
    one = torch.autograd.grad(loss * 0.5, (h, w), retain_graph=True)
    two = torch.autograd.grad(loss, (h, w))
    # a factor applied to gradients that are rounded already: one more rounding
    within(one[0], 0.5 * dh, edh + U[dtype] * dh.abs() + 2.0 ** -24, "half the loss")
    within(two[0], dh, edh, "dh again")
    within(two[1], dw, edw, "dw again")
    only_h = torch.autograd.grad(lce(h, w.detach(), y), h)[0]
    only_w = torch.autograd.grad(lce(h.detach(), w, y), w)[0]
    assert torch.equal(only_h, two[0]) and torch.equal(only_w, two[1])


def test_gradient_matches_differences():
    h, w, y = make(90, 640, 80, "f32", seed=9, ignored=0.2)
    h.requires_grad_(True)
    w.requires_grad_(True)
    lce(h, w, y, label_smoothing=0.05).backward()
    g = torch.Generator().manual_seed(1)
    dh = torch.randn(h.shape, generator=g).cuda()
    dw = torch.randn(w.shape, generator=g).cuda() * 0.1
    eps = 2.0 ** -7
    with torch.no_grad():
        a = lce(h + eps * dh, w + eps * dw, y, label_smoothing=0.05)
        b = lce(h - eps * dh, w - eps * dw, y, label_smoothing=0.05)
        slope = (float(a) - float(b)) / (2 * eps)
        want = float((h.grad.double() * dh.double()).sum() + (w.grad.double() * dw.double()).sum())
    # the third derivative of the loss along the line: |h dw + dh w| is about 3 per logit,
    # so eps^2 / 6 * 3^3 * 2; and float32 losses of about 6 over 2 eps
    assert abs(slope - want) <= eps ** 2 / 6 * 54 + 8 * F * 6 / (2 * eps)


def test_two_calls_are_bit_identical_and_streams_are_kept():
    h, w, y = make(400, 3000, 256, "bf16", seed=10, ignored=0.25)

    def both():
        hh, ww = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = lce(hh, ww, y)
        return (loss.detach(),) + torch.autograd.grad(loss, (hh, ww))

    first = both()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = both()
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_a_captured_call_replays():
    h, w, y = make(200, 1500, 128, "bf16", seed=11, ignored=0.25)
    loss = torch.zeros((), device="cuda")

    def run():
        with torch.no_grad():
            return lce(h, w, y)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = run()
    for k in range(4):
        h.copy_(make(200, 1500, 128, "bf16", seed=20 + k)[0])
        y[k] = IGNORE
        eager = run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, eager)


def test_indices_past_32_bits():
    """Kept values of more than 2^31 elements, and a weight of more than 2^32 bytes."""
    n, v, d = 8192, 270000, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    h = torch.randn(n, d, device="cuda", generator=g).bfloat16().requires_grad_(True)
    w = (torch.randn(v, d, device="cuda", generator=g) * 0.1).bfloat16().requires_grad_(True)
    y = torch.randint(0, v, (n,), device="cuda", generator=g)
    loss = lce(h, w, y, workspace_limit=8 << 30)
    dh, dw = torch.autograd.grad(loss, (h, w))
    part = torch.tensor([0, 1, 4095, 4096, 7000, 8000, 8190, 8191], device="cuda")
    ref = definition(h.detach()[part], w.detach(), y[part], "bf16", row_grad=torch.full((8,), 1.0 / n, device="cuda"))
    within(dh[part], ref[2], ref[3], "dh")
    # the last columns' rows of dW from all positions: p needs every position's lse
    with torch.no_grad():
        lse = torch.cat([torch.logsumexp(torch.mm(h.detach()[i:i + 512].double(), w.detach().double().t()), 1)
                         for i in range(0, n, 512)])
        cols = torch.tensor([0, 131071, 262143, 262144, 269999], device="cuda")
        lg = torch.mm(h.detach().double(), w.detach().double()[cols].t())
        p = (lg - lse[:, None]).exp()
        hit = (y[:, None] == cols[None]).double()
        want = torch.mm((p - hit).t() / n, h.detach().double())
        size = torch.mm((p * 0.012 + hit * 0.004).t() / n, h.detach().double().abs())
    within(dw[cols], want, size + 2.0 ** -8 * want.abs(), "dw")
    del h, w, dh, dw
    n, v, d = 3, 1000003, 2304
    w = torch.empty(v, d, dtype=torch.bfloat16, device="cuda").normal_(generator=g).mul_(0.02)
    h = torch.randn(n, d, device="cuda", generator=g).bfloat16()
    y = torch.tensor([0, v - 1, 970001], device="cuda")
    got = lce(h, w, y, reduction="none")
    lg = torch.cat([torch.mm(h.float(), w[i:i + 100000].float().t()) for i in range(0, v, 100000)], 1).double()
    want = torch.logsumexp(lg, 1) - lg.gather(1, y[:, None])[:, 0]
    # float32 sums on both sides
    assert float((got.double() - want).abs().max()) <= 2 * (d + 2) * F * float(h.float().abs().max()) * 0.02 * d


def test_refusals():
    h, w, y = make(8, 30, 16, "bf16")
    with pytest.raises(TypeError):
        lce([1.0], w, y)
    with pytest.raises(ValueError, match="CUDA"):
        lce(h.cpu(), w, y)
    with pytest.raises(ValueError, match="dtype"):
        lce(h, w.float(), y)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        lce(h.double(), w.double(), y)
    with pytest.raises(ValueError, match="targets of shape"):
        lce(h, w, y[:7])
    with pytest.raises(ValueError, match="int64 or int32"):
        lce(h, w, y.float())
    with pytest.raises(ValueError, match="width"):
        lce(h, w[:, :15], y)
    with pytest.raises(ValueError, match="2D"):
        lce(h, w[0], y)
    with pytest.raises(ValueError, match="non-empty"):
        lce(h, w[:0], y)
    with pytest.raises(ValueError, match="reduction"):
        lce(h, w, y, reduction="max")
    with pytest.raises(ValueError, match="label_smoothing"):
        lce(h, w, y, label_smoothing=1.5)
    with pytest.raises(ValueError, match="workspace_limit"):
        lce(h, w, y, workspace_limit=0)
