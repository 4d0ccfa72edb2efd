"""rms_norm, rms_norm_quantized and dropout against their definitions in float64, and their calls.

Error bounds (u: half the spacing of the dtype at 1, f = 2^-24, W the width):

* the factors of dropout are exact but for one rounding, and so is the sum: s is off by
  es = 3 f (|x| m / (1 - p) + |residual|);
* r is formed in float64 from s and rounded: relative max(es / |s|) at most, so a row's r is off
  by 2 f + max es / rms(s), rms the row's root mean square (with eps);
* y = s r w: three roundings and those, then u;
* backward reads s rounded to the dtype (u |s| more; none in float32): n = s r is off by
  en = r (u |s| + es) + |n| (the error of r + 2 f); mean(g n) by the mean of its terms' errors
  and (W / 8 + 16) f of the mean of |g n| (eight partial sums a lane, then a tree); ds by the sum of
  those, and u of its own;
* dw is a sum over R rows: its terms' errors, R f of their sizes, and u;
* where a result is rounded to float16, half its subnormal spacing, 2^-25, more."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}
F = 2.0 ** -24
SEED = 0x123456789ABCDEF


def philox(block, offset, seed):
    """Philox4x32-10 in Python integers: the eight 16-bit values of a block."""
    m = 0xFFFFFFFF
    c = [block & m, block >> 32, offset & m, offset >> 32]
    k = [seed & m, (seed >> 32) & m]
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & m, (a >> 32) ^ c[3] ^ k[1], a & m]
        k = [(k[0] + 0x9E3779B9) & m, (k[1] + 0xBB67AE85) & m]
    return [w >> s & 0xFFFF for w in c for s in (0, 16)]


def kept(n, p, seed=SEED, offset=0):
    """Factors of n elements, float64 on the CPU."""
    cut = round(p * 65536)
    u = [x for b in range(-(-n // 8)) for x in philox(b, offset, seed)][:n]
    return (torch.tensor(u) >= cut).double() * (65536.0 / (65536 - cut) if cut < 65536 else 0.0)


def make(dtype, shape, seed=0):
    g = torch.Generator().manual_seed(seed + 31 * shape[-1] + shape[0])
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    res = 3.0 * r(*shape)
    res[..., ::7] *= 8.0
    return tuple(t.to(DT[dtype]).cuda() for t in (r(*shape), res, 1.0 + 0.3 * r(shape[-1]), r(*shape), r(*shape)))


def definition(dtype, x, res, w, dy, ds, eps, factors=None):
    """((y, s, dx, dres, dw), their bounds), float64."""
    u, tiny = U[dtype], TINY[dtype]
    rounded = 0.0 if dtype == "f32" else u
    x, w, dy = x.double(), w.double(), dy.double()
    keep = torch.ones_like(x) if factors is None else factors.to(x.device).view(x.shape)
    s = x * keep
    es = 3 * F * s.abs()
    if res is not None:
        s = s + res.double()
        es = 3 * F * ((x * keep).abs() + res.double().abs())
    elif factors is None:
        es = es * 0
    width = x.shape[-1]
    rms = (s.square().mean(-1, keepdim=True) + eps).sqrt()
    r = 1 / rms
    er = 2 * F + es.amax(-1, keepdim=True) / rms  # relative
    n = s * r
    y = n * w
    ey = (es * r * w.abs()) + y.abs() * (er + 3 * F + u) + tiny
    en = r * (rounded * s.abs() + es) + n.abs() * (er + 2 * F)
    g = dy * w
    dot = (g * n).mean(-1, keepdim=True)
    edot = (g.abs() * en).mean(-1, keepdim=True) + (width / 8 + 16) * F * (g * n).abs().mean(-1, keepdim=True)
    d = r * (g - n * dot)
    ed = r * (en * dot.abs() + n.abs() * edot + 6 * F * (g.abs() + (n * dot).abs())) + d.abs() * er
    if ds is not None:
        d = d + ds.double()
        ed = ed + 2 * F * (d.abs() + ds.double().abs())
    dx, edx = d * keep, (ed + 2 * F * d.abs()) * keep
    rows = x.numel() // width
    flat = lambda t: t.reshape(-1, width)  # noqa: E731
    dw = flat(dy * n).sum(0)
    edw = flat(dy.abs() * (en + 2 * F * n.abs())).sum(0) + (rows + 4) * F * flat((dy * n).abs()).sum(0)
    fin = lambda v, e: e * (1 + u) + u * v.abs() + tiny  # noqa: E731
    return (y, s, dx, d, dw), (ey, fin(s, es), fin(dx, edx), fin(d, ed), fin(dw, edw))


def within(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, what
    assert bool(torch.isfinite(got).all()), what
    bad = (got - want).abs() > bound
    assert not bool(bad.any()), "{}: {} of {} outside, worst {:.3g} of its bound".format(
        what, int(bad.sum()), bad.numel(), float(((got - want).abs() / bound.clamp(min=1e-300)).max()))


def call(x, res, w, dy, ds, **kw):
    from gefen_amd import rms_norm

    leaves = [t.detach().requires_grad_(True) for t in (x, res, w) if t is not None]
    if res is None:
        y = rms_norm(leaves[0], leaves[1], **kw)
        dx, dw = torch.autograd.grad(y, leaves, grad_outputs=dy)
        return y.detach(), None, dx, None, dw
    y, s = rms_norm(leaves[0], leaves[2], residual=leaves[1], **kw)
    dx, dr, dw = torch.autograd.grad((y, s), leaves, grad_outputs=(dy, ds))
    return y.detach(), s.detach(), dx, dr, dw


NAMES = ("y", "sum", "dx", "dresidual", "dweight")
SHAPES = [(1, 1), (3, 7), (48, 96), (5, 511), (9, 512), (2, 513), (37, 1001), (4, 1024), (3, 1025), (130, 2048),
          (7, 2049), (20, 4096), (3, 4100), (2, 8192), (3, 8193), (2, 16384), (3, 16385), (2, 32768), (700, 40),
          (2, 3, 65)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("mode", ["plain", "residual", "dropout"])
def test_results_and_gradients_match_the_definition(dtype, shape, mode):
    x, res, w, dy, ds = make(dtype, shape)
    kw, factors = {"eps": 1e-5}, None
    if mode == "plain":
        res = ds = None
    if mode == "dropout":
        if x.numel() > 20000:
            pytest.skip("the generator in Python integers takes too long")
        kw.update(dropout=0.3, seed=SEED, offset=7)
        factors = kept(x.numel(), 0.3, offset=7)
    got = call(x, res, w, dy, ds, **kw)
    for a, b, e, name in zip(got, *definition(dtype, x, res, w, dy, ds, 1e-5, factors), NAMES):
        if a is not None:
            within(a, b, e, name)
    with torch.no_grad():
        from gefen_amd import rms_norm

        again = rms_norm(x, w, residual=res, **kw)
    assert torch.equal(again if res is None else again[0], got[0])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_many_rows(dtype):
    """More rows than the workgroups of a launch, so that each takes several."""
    for shape in ((9001, 24), (3000, 1100)):
        x, res, w, dy, ds = make(dtype, shape)
        got = call(x, res, w, dy, ds)
        for a, b, e, name in zip(got, *definition(dtype, x, res, w, dy, ds, 1e-6), NAMES):
            within(a, b, e, name)
        assert all(torch.equal(a, b) for a, b in zip(got, call(x, res, w, dy, ds)))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("name", ["float8_e4m3fn", "float8_e5m2"])
def test_eight_bits(dtype, name):
    """Each value is the nearest of the format to y / scale: within half a step (2^-4 or 2^-3 of the
    value, or half the format's smallest spacing), and y's own error."""
    from gefen_amd import rms_norm_quantized

    fmt = getattr(torch, name)
    most, half_step, tiny = (448.0, 2.0 ** -4, 2.0 ** -10) if "e4m3" in name else (57344.0, 2.0 ** -3, 2.0 ** -17)
    for shape in SHAPES:
        for res in (True, False):
            x, r, w, dy, ds = make(dtype, shape)
            r = r if res else None
            with torch.no_grad():
                q, scales, *s = rms_norm_quantized(x, w, residual=r, eps=1e-5, dtype=fmt)
            (y, total, *_), (_, es, *_) = definition("f32", x, r, w, dy, None, 1e-5)
            assert q.dtype == fmt and q.shape == x.shape and scales.shape == x.shape[:-1] and len(s) == res
            c = y.abs().amax(-1) / most
            err = 64 * F
            assert bool(((scales.double() - c).abs() <= err * c).all())
            back = q.double() * scales.double()[..., None]
            assert bool(((back - y).abs() <= half_step * y.abs() + (tiny + err * most) * c[..., None]).all())
            # and the rounding is the format's own, to nearest even, of the float32 quotient
            if s:
                within(s[0], total, 3 * F * total.abs() + U[dtype] * total.abs() + 24 * F + TINY[dtype], "sum")


def test_eight_bits_of_edges():
    from gefen_amd import rms_norm_quantized

    x = torch.zeros(4, 40, device="cuda")
    x[1, 3] = 1.0
    x[2, 5] = math.nan
    x[3, 7] = math.inf
    with torch.no_grad():
        q, c = rms_norm_quantized(x, torch.ones(40, device="cuda"))
    q = q.float()
    assert not bool(q[0].any()) and float(c[0]) == 0.0
    assert float(q[1, 3]) == 448.0 and not bool(q[1, :3].any())
    assert bool(torch.isnan(q[2] * c[2]).all()) and not bool(torch.isfinite(q[3] * c[3]).all())
    # every value of the format comes out where it went in: y = x, the row's rms held at 1
    for fmt in (torch.float8_e4m3fn, torch.float8_e5m2):
        bits = torch.arange(256, dtype=torch.int16).to(torch.uint8).cuda().view(fmt).float()
        vals = bits[torch.isfinite(bits)]
        row = vals / float(vals.abs().max())
        w = torch.full((row.numel(),), float(row.square().mean().sqrt()), device="cuda")
        with torch.no_grad():
            q, c = rms_norm_quantized(row[None], w, eps=0.0, dtype=fmt)
        near = (q[0].float() - vals).abs() <= 2.0 ** -20 * vals.abs()
        assert bool(near.all())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0, 2.0 ** -16, 0.9999])
def test_dropout(dtype, p):
    from gefen_amd import dropout

    for n in (1, 7, 8, 9, 1000, 4099):
        x, res, _, dy, _ = make(dtype, (n,), seed=3)
        m = kept(n, p, offset=(5 << 32) + 2).cuda()
        a, b = x.detach().requires_grad_(True), res.detach().requires_grad_(True)
        y = dropout(a, p, SEED, offset=(5 << 32) + 2, residual=b)
        da, db = torch.autograd.grad(y, (a, b), grad_outputs=dy)
        u, tiny = U[dtype], TINY[dtype]
        want = x.double() * m + res.double()
        within(y.detach(), want, u * want.abs() + 3 * F * ((x.double() * m).abs() + res.double().abs()) + tiny, "y")
        for got, src in ((da, dy), (dropout(x, p, SEED, offset=(5 << 32) + 2), x)):
            want = src.double() * m
            fits = want.abs() < torch.finfo(DT[dtype]).max
            bound = (u + 4 * F) * want.abs() + tiny
            assert bool(((got.double() - want).abs() <= bound)[fits].all())
        assert torch.equal(db, dy)


def test_dropout_keeps_its_share_and_differs_by_seed_and_offset():
    """Of n elements (1 - p) n are kept, within 6 standard deviations."""
    from gefen_amd import dropout

    n = 1 << 22
    ones = torch.ones(n, device="cuda")
    masks = [dropout(ones, 0.25, s, offset=o) > 0 for s, o in ((1, 0), (2, 0), (1, 1), (1 + (1 << 40), 0), (1, 1 << 40))]
    for i, m in enumerate(masks):
        assert abs(int(m.sum()) - 0.75 * n) <= 6 * math.sqrt(n * 0.25 * 0.75)
        for o in masks[:i]:  # independent: both kept in (1 - p)^2
            q = 0.75 * 0.75
            assert abs(int((m & o).sum()) - q * n) <= 6 * math.sqrt(n * q * (1 - q))
    assert torch.equal(dropout(ones, 0.25, 1) > 0, masks[0])


def test_seeds_of_all_kinds():
    from gefen_amd import dropout

    x = torch.ones(5000, device="cuda")
    for value in (0, 1, -1, (1 << 63) - 1, -(1 << 63)):
        t = torch.tensor(value, dtype=torch.int64, device="cuda")
        assert torch.equal(dropout(x, 0.5, value), dropout(x, 0.5, t))
        assert torch.equal(dropout(x, 0.5, value), dropout(x, 0.5, t.view(1)))
        assert torch.equal(dropout(x, 0.5, value), dropout(x, 0.5, value % (1 << 64)))


def test_far_elements_of_a_large_tensor():
    """Elements past 2^32 take their own place of the generator."""
    from gefen_amd import dropout

    n = (1 << 32) + 64
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = dropout(x, 0.5, SEED)
    del x
    u = [v for b in range((1 << 32) // 8, n // 8) for v in philox(b, 0, SEED)]
    assert y[1 << 32:].tolist() == [2.0 if v >= 32768 else 0.0 for v in u]


def test_what_is_dropped_counts_as_zero():
    from gefen_amd import dropout, rms_norm

    x, res, w, dy, ds = make("f32", (4, 600))
    m = kept(2400, 0.4).view(4, 600).cuda() > 0
    bad = torch.where(m, x, torch.full_like(x, math.nan))
    assert torch.equal(dropout(bad, 0.4, SEED, residual=res), dropout(x, 0.4, SEED, residual=res))
    a, b = (call(t, res, w, dy, ds, dropout=0.4, seed=SEED) for t in (bad, x))
    assert all(torch.equal(i, j) for i, j in zip(a, b))
    y, s = rms_norm(x, w, residual=res, dropout=0.4, seed=SEED)
    assert torch.equal(s, dropout(x, 0.4, SEED, residual=res))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_strides_orders_and_alignment(dtype):
    x, res, w, dy, ds = make(dtype, (6, 9, 70))
    kw = {"dropout": 0.2, "seed": SEED}
    want = call(x, res, w, dy, ds, **kw)
    from gefen_amd import dropout

    want_drop = dropout(x, 0.2, SEED, residual=res)

    def odd(t):  # one element off any alignment, rows of 73
        buf = torch.full((t.numel() // 70 * 73 + 1,), math.nan, dtype=t.dtype, device="cuda")
        view = buf[1:].view(*t.shape[:-1], 73)[..., :70] if t.dim() > 1 else buf[1:71]
        view.copy_(t)
        return view

    permuted = lambda t: t.transpose(0, -1).contiguous().transpose(0, -1)  # noqa: E731
    for f in (odd, permuted, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1) if t.dim() > 1 else t):
        got = call(f(x), f(res), odd(w), f(dy), f(ds), **kw)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(dropout(f(x), 0.2, SEED, residual=f(res)), want_drop)
    row = torch.ones(70, dtype=x.dtype, device="cuda")
    a = call(x, res, w, row.expand(x.shape), row.expand(x.shape))
    b = call(x, res, w, torch.ones_like(x), torch.ones_like(x))
    assert all(torch.equal(i, j) for i, j in zip(a, b))


def test_values_whose_squares_leave_the_range():
    from gefen_amd import rms_norm

    for scale in (1e30, 1e-30):
        x, _, w, _, _ = make("f32", (3, 200))
        with torch.no_grad():
            got = rms_norm(x * scale, w, eps=0.0)
        want = definition("f32", x * scale, None, w, x, None, 0.0)[0][0]
        within(got, want, 16 * F * want.abs(), "y")


def test_only_some_gradients_are_wanted():
    from gefen_amd import rms_norm

    x, res, w, dy, ds = make("bf16", (30, 200))
    for kw in ({}, {"dropout": 0.1, "seed": 4}):
        _, _, dx, dr, dw = call(x, res, w, dy, ds, **kw)
        want = dict(zip("xrw", (dx, dr, dw)))
        for names in ("x", "r", "w", "xr", "xw", "rw"):
            t = {n: v.detach().requires_grad_(n in names) for n, v in zip("xrw", (x, res, w))}
            y, s = rms_norm(t["x"], t["w"], residual=t["r"], **kw)
            torch.autograd.backward((y, s), (dy, ds))
            for n in "xrw":
                assert (t[n].grad is None) == (n not in names)
                assert n not in names or torch.equal(t[n].grad, want[n])
    # one of the two results only
    a, b = (t.detach().requires_grad_(True) for t in (x, res))
    y, s = rms_norm(a, w, residual=b)
    got = torch.autograd.grad(s, (a, b), grad_outputs=ds, retain_graph=True)
    assert torch.equal(got[0], ds) and torch.equal(got[1], ds)
    got = torch.autograd.grad(y, (a,), grad_outputs=dy)
    assert torch.equal(got[0], call(x, res, w, dy, torch.zeros_like(ds))[2])


def test_gradients_that_are_equal_do_not_share_in_grad():
    from gefen_amd import clip_grad_norm_, rms_norm

    x, res, w, dy, ds = (t.requires_grad_(i < 3) for i, t in enumerate(make("f32", (8, 64))))
    torch.autograd.backward(rms_norm(x, w, residual=res), (dy, ds))
    before = x.grad.clone()
    assert torch.equal(x.grad, res.grad)
    norm = clip_grad_norm_([x, res, w], 0.5)
    assert torch.allclose(x.grad, before * (0.5 / (norm + 1e-6)), rtol=4 * F, atol=0)
    assert torch.equal(x.grad, res.grad)


def test_gradients_agree_with_differences():
    """Along a direction: the difference quotient's truncation is that of the definition's own, its
    rounding the results' bounds at both ends."""
    x, res, w, dy, ds = make("f32", (5, 130), seed=9)
    kw = {"dropout": 0.25, "seed": SEED}
    m = kept(650, 0.25)
    grads = dict(zip(NAMES, call(x, res, w, dy, ds, **kw)))
    wants = dict(zip(NAMES, zip(*definition("f32", x, res, w, dy, ds, 1e-6, m))))
    from gefen_amd import rms_norm

    h = 2.0 ** -8
    g = torch.Generator(device="cuda").manual_seed(3)
    for i, name in enumerate(("dx", "dresidual", "dweight")):
        step = h * torch.sign(torch.randn((x, res, w)[i].shape, device="cuda", generator=g))
        ends, exact, rounding = [], [], 0.0
        for sign in (1, -1):
            ts = [x, res, w]
            ts[i] = ts[i] + sign * step
            with torch.no_grad():
                y, s = rms_norm(ts[0], ts[2], residual=ts[1], **kw)
            ends.append(float((y.double() * dy.double()).sum() + (s.double() * ds.double()).sum()))
            (ty, tsum, *_), (ey, es, *_) = definition("f32", *ts, dy, ds, 1e-6, m)
            exact.append(float((ty * dy.double()).sum() + (tsum * ds.double()).sum()))
            rounding += float((ey * dy.double().abs()).sum() + (es * ds.double().abs()).sum())
        slope = float((grads[name].double() * 2 * step.double()).sum())
        true_slope = float((wants[name][0] * 2 * step.double()).sum())
        allowed = abs(exact[0] - exact[1] - true_slope) + rounding + float((wants[name][1] * 2 * h).sum())
        assert abs(ends[0] - ends[1] - slope) <= allowed


def test_a_captured_step_takes_the_seed_of_each_replay():
    from gefen_amd import dropout, rms_norm

    x, res, w, dy, ds = make("bf16", (300, 200))
    seed = torch.tensor(11, dtype=torch.int64, device="cuda")
    leaves = [t.detach().requires_grad_(True) for t in (x, res, w)]

    def step():
        y, s = rms_norm(leaves[0], leaves[2], residual=leaves[1], dropout=0.2, seed=seed, offset=3)
        return (y, s, dropout(y.detach(), 0.3, seed, offset=4)) + torch.autograd.grad((y, s), leaves, grad_outputs=(dy, ds))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    last = None
    for k in range(4):
        seed.fill_(11 + k)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.detach(), b.detach()) for a, b in zip(got, step()))
        assert last is None or not torch.equal(last, got[1])
        last = got[1].detach().clone()


def test_a_seed_changed_before_backward_is_noticed():
    from gefen_amd import dropout

    x = torch.ones(64, device="cuda", requires_grad=True)
    seed = torch.tensor(5, dtype=torch.int64, device="cuda")
    y = dropout(x, 0.5, seed)
    seed += 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_empty_tensors():
    from gefen_amd import dropout, rms_norm, rms_norm_quantized

    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    y, s = rms_norm(x, w, residual=x)
    (y.sum() + s.sum()).backward()
    assert x.grad.shape == (0, 16) and not bool(w.grad.any())
    with torch.no_grad():
        q, c = rms_norm_quantized(x, w)
    assert q.shape == (0, 16) and c.shape == (0,)
    assert dropout(x, 0.5, 1).shape == (0, 16)


def test_refusals_on_the_device():
    from gefen_amd import dropout, rms_norm, rms_norm_quantized

    x, w = torch.ones(4, 16, device="cuda"), torch.ones(16, device="cuda")
    seed = torch.tensor(1, device="cuda")
    calls = [lambda: rms_norm(x, w[:8]), lambda: rms_norm(x, w[None]), lambda: rms_norm(x, w.half()),
             lambda: rms_norm(x, w, residual=x[:2]), lambda: rms_norm(x, w, residual=x.half()),
             lambda: rms_norm(x, w.cpu()), lambda: rms_norm(x.double(), w.double()), lambda: rms_norm(x, w, eps=-1.0),
             lambda: rms_norm(x, w, eps=math.nan), lambda: rms_norm(x, w, eps=math.inf),
             lambda: rms_norm(x, w, dropout=0.1, seed=1), lambda: rms_norm(x, w, residual=x, dropout=0.1),
             lambda: rms_norm(x, w, residual=x, dropout=1.5, seed=1), lambda: rms_norm(x[:, :0], w[:0]),
             lambda: rms_norm(torch.ones(32769, device="cuda"), torch.ones(32769, device="cuda")),
             lambda: rms_norm(x[0, 0], w), lambda: rms_norm_quantized(x, w, dtype=torch.int8),
             lambda: rms_norm_quantized(x.clone().requires_grad_(True), w), lambda: dropout(x, -0.1, 1),
             lambda: dropout(x, math.nan, 1), lambda: dropout(x, 0.1, 1 << 64), lambda: dropout(x, 0.1, 1, offset=-1),
             lambda: dropout(x, 0.1, seed.cpu()), lambda: dropout(x, 0.1, seed.int()),
             lambda: dropout(x, 0.1, torch.ones(2, dtype=torch.int64, device="cuda")),
             lambda: dropout(x, 0.1, 1, residual=x[:2]), lambda: dropout(x.int(), 0.1, 1)]
    for k, f in enumerate(calls):
        with pytest.raises(ValueError):
            f()
            raise AssertionError("call {} was taken".format(k))
    for f in (lambda: dropout(x, 0.1, 1.5), lambda: dropout(x, 0.1, True), lambda: rms_norm(x, None),
              lambda: dropout([1.0], 0.1, 1)):
        with pytest.raises(TypeError):
            f()
