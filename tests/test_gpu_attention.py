"""attention against its definition in float64, what must not reach a result, and its calls.

Error bounds, element by element (u: half the spacing of the operands' dtype at 1, 2^-8
for bf16, 2^-11 for f16, 2^-24 for f32; f = 2^-24; D the width, n the keys, m the rows that
share a key head):

* a score is a float32 sum of D exact products, times a rounded constant: off by at most
  es = (D + 4) f sum |q k| scale; E is the largest of a row;
* a probability is exp(score - L): relative delta = 2 E + (2 n + 32) f + 8 f max |S| (both
  sides of the difference, the sum of n terms, exp and log at a few f, their arguments'
  rounding), and u more where it is rounded on its way into a product (float32: not at all);
  float16 keeps it times 2^6 (2^14 backward) with a spacing of 2^-24, half of that the error,
  against a sum that is at least 2^6: 2^-31, 2^-39 backward;
* a product over n terms adds (n + 4) f of the sum of their sizes, a result u of its own and
  float16 half its subnormal spacing 2^-25;
* D_i is formed of the rounded output: its error is that of the output times |dO|, and a sum;
* dS = P (dP - D) has the errors of its factors, u of its own, and in float16 2^-25 of a
  spacing at 2^14 of the bound B = 4 |dO_i| max |v_j| (a power of two at most twice
  2 |dO_i| max |v_j|): 2^-39 B, with the largest row's |dO| for dK."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
F = 2.0 ** -24


def attention(*a, **k):
    from gefen_amd import attention as f

    return f(*a, **k)


def make(dtype, b, sq, sk, h, hk, d, seed=0, grad=1.0):
    g = torch.Generator().manual_seed(seed + 131 * sq + 17 * sk + d)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    return tuple(x.to(DT[dtype]).cuda() for x in (1.5 * r(b, sq, h, d), r(b, sk, hk, d), r(b, sk, hk, d),
                                                  grad * r(b, sq, h, d)))


def visible(b, sq, sk, causal=False, lengths=None, offsets=None):
    """[b, sq, sk] truth values."""
    i, j = torch.arange(sq)[:, None], torch.arange(sk)[None]
    m = torch.ones(b, sq, sk, dtype=torch.bool)
    if causal:
        m &= (j <= i + sk - sq)
    if lengths is not None:
        m &= (j < torch.tensor(lengths)[:, None, None])
    if offsets is not None:
        of = torch.full((sq,), -1)
        for s, (a, e) in enumerate(zip(offsets, offsets[1:])):
            of[a:e] = s
        m &= (of[:, None] == of[None]) & (of[:, None] >= 0)
    return m.cuda()


def definition(q, k, v, go, seen, dtype, scale=None):
    """(out, dq, dk, dv) and their bounds, float64, of [b, s, h, d] operands."""
    b, sq, h, d = q.shape
    sk, hk = k.shape[1:3]
    grp = h // hk
    scale = d ** -0.5 if scale is None else scale
    u = U[dtype]
    up = 0.0 if dtype == "f32" else u
    half = dtype == "f16"
    fold = lambda t: t.double().transpose(1, 2).reshape(b * hk, -1, d)  # noqa: E731
    q, go, k, v = (fold(t) for t in (q, go, k, v))
    seen = seen[:, None].expand(b, h, sq, sk).reshape(b * hk, grp * sq, sk)
    T = lambda t: t.transpose(1, 2).contiguous()  # noqa: E731
    zero = torch.zeros((), dtype=torch.float64, device=q.device)
    mask = lambda t: torch.where(seen, t, zero)  # noqa: E731
    any_key = seen.any(2, keepdim=True)
    s = torch.bmm(q, T(k)) * scale
    es = mask((d + 4) * F * scale * torch.bmm(q.abs(), T(k).abs()))
    e_row = es.amax(2, keepdim=True) if sk else zero
    smax = mask(s.abs()).amax(2, keepdim=True) if sk else zero
    top = torch.where(seen, s, zero - math.inf).amax(2, keepdim=True) if sk else zero
    top = torch.where(any_key, top, zero)
    p = mask((s - top).exp())
    p = p / torch.where(any_key, p.sum(2, keepdim=True), zero + 1)
    n, m = sk, sq * grp
    delta = 2 * e_row + (2 * n + 32) * F + 8 * F * smax
    o = torch.bmm(p, v)
    a = torch.bmm(p, v.abs())
    eo = a * (delta + up + (n + 4) * F) + u * o.abs()
    if half:
        eo = eo + 2.0 ** -31 * torch.bmm(seen.double(), v.abs()) + 2.0 ** -25
    dv = torch.bmm(T(p), go)
    edv = torch.bmm(T(p * (delta + up)), go.abs()) + (m + 4) * F * torch.bmm(T(p), go.abs()) + u * dv.abs()
    dp = torch.bmm(go, T(v))
    edp = (d + 2) * F * torch.bmm(go.abs(), T(v).abs())
    big = (go * o).sum(2, keepdim=True)
    ebig = (go.abs() * eo).sum(2, keepdim=True) + (d + 2) * F * (go * o).abs().sum(2, keepdim=True)
    ds = p * (dp - big)
    eds = p * (delta * (dp - big).abs() + edp + ebig + 4 * F * (dp.abs() + big.abs())) + up * ds.abs()
    eds_k = eds
    if half:
        vmax = v.norm(dim=2).amax(1)[:, None, None] if sk else zero
        bound = 4 * go.norm(dim=2, keepdim=True) * vmax
        edv = edv + 2.0 ** -39 * torch.bmm(T(seen.double()), go.abs()) + 2.0 ** -25
        eds, eds_k = eds + mask(2.0 ** -39 * bound), eds + mask(2.0 ** -39 * bound.amax(1, keepdim=True))
    dq, dk = scale * torch.bmm(ds, k), scale * torch.bmm(T(ds), q)
    edq = scale * (torch.bmm(eds, k.abs()) + (n + 6) * F * torch.bmm(ds.abs(), k.abs())) + u * dq.abs()
    edk = scale * (torch.bmm(T(eds_k), q.abs()) + (m + 6) * F * torch.bmm(T(ds.abs()), q.abs())) + u * dk.abs()
    if half:
        edq, edk = edq + 2.0 ** -25, edk + 2.0 ** -25
    back = lambda t, heads: t.view(b, heads, -1, d).transpose(1, 2)  # noqa: E731
    return ([back(o, h), back(dq, h), back(dk, hk), back(dv, hk)],
            [back(eo, h), back(edq, h), back(edk, hk), back(edv, hk)])


def within(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, what
    assert bool(torch.isfinite(got).all()), what
    bad = (got - want).abs() > bound
    assert not bool(bad.any()), "{}: {} of {} outside, worst {:.3g} of its bound".format(
        what, int(bad.sum()), bad.numel(), float(((got - want).abs() / bound.clamp(min=1e-300)).max()))


NAMES = ("out", "dquery", "dkey", "dvalue")


def call(q, k, v, go, **kw):
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = attention(q, k, v, **kw)
    return (out.detach(),) + torch.autograd.grad(out, (q, k, v), grad_outputs=go)


def compare(dtype, q, k, v, go, seen, scale=None, **kw):
    got = call(q, k, v, go, **({} if scale is None else {"scale": scale}), **kw)
    want, bounds = definition(q, k, v, go, seen, dtype, scale)
    for x, w, e, name in zip(got, want, bounds, NAMES):
        within(x, w, e, name)
    with torch.no_grad():
        again = attention(q, k, v, **({} if scale is None else {"scale": scale}), **kw)
    assert torch.equal(again, got[0])


SIZES = [(1, 1, 1, 1, 1, 1), (2, 1, 7, 4, 2, 8), (1, 5, 3, 3, 1, 33), (3, 19, 19, 4, 4, 24), (2, 64, 64, 2, 2, 64),
         (1, 65, 63, 6, 2, 80), (2, 127, 200, 5, 5, 96), (1, 129, 129, 8, 1, 128), (1, 300, 333, 4, 2, 127),
         (2, 1, 1003, 8, 2, 128), (1, 777, 40, 2, 1, 17), (1, 520, 520, 3, 3, 64)]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("b,sq,sk,h,hk,d", SIZES)
def test_results_and_gradients_match_the_definition(dtype, b, sq, sk, h, hk, d, causal):
    q, k, v, go = make(dtype, b, sq, sk, h, hk, d)
    compare(dtype, q, k, v, go, visible(b, sq, sk, causal), causal=causal)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_key_lengths(dtype, causal, index):
    lengths = [0, 1, 64, 65, 150, 131]
    q, k, v, go = make(dtype, 6, 140, 150, 4, 2, 40)
    compare(dtype, q, k, v, go, visible(6, 140, 150, causal, lengths), causal=causal,
            key_lengths=torch.tensor(lengths, dtype=index, device="cuda"))


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("offsets", [[0, 300], [0, 1, 2, 65, 65, 200, 300], [10, 90, 91, 290], [0, 0, 0],
                                     [7]])
def test_packed_sequences(dtype, causal, index, offsets):
    q, k, v, go = make(dtype, 1, 300, 300, 4, 2, 64)
    seen = visible(1, 300, 300, causal, offsets=offsets)
    got = call(q[0], k[0], v[0], go[0], causal=causal, offsets=torch.tensor(offsets, dtype=index, device="cuda"))
    want, bounds = definition(q, k, v, go, seen, dtype)
    for x, w, e, name in zip(got, want, bounds, NAMES):
        within(x[None], w, e, name)
        inside = torch.zeros(300, dtype=torch.bool)
        inside[offsets[0]:offsets[-1]] = True
        assert not bool(x[~inside.cuda()].any()), name


def test_lengths_out_of_range_are_taken_into_it():
    q, k, v, go = make("bf16", 3, 20, 30, 2, 2, 16)
    got = call(q, k, v, go, key_lengths=torch.tensor([-5, 1 << 40, 30], device="cuda"))
    want = call(q, k, v, go, key_lengths=torch.tensor([0, 30, 30], device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # offsets past the tokens, and descending ones, stay in bounds
    for offsets in ([0, 10, 1 << 40], [-3, 12, 20], [20, 5, 0], [0, 15, 5, 20]):
        out = call(q[0], q[1], q[2], go[0], offsets=torch.tensor(offsets, device="cuda"))
        assert all(bool(torch.isfinite(t).all()) for t in out)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_scales(dtype):
    q, k, v, go = make(dtype, 1, 70, 70, 2, 1, 32)
    for scale in (0.0, 0.01, 1.0):
        compare(dtype, q, k, v, go, visible(1, 70, 70, True), scale=scale, causal=True)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_rows_without_keys_and_no_keys_at_all(dtype):
    q, k, v, go = make(dtype, 2, 9, 4, 2, 1, 16)  # causal: the first five queries see nothing
    out, dq, dk, dv = call(q, k, v, go, causal=True)
    assert not bool(out[:, :5].any()) and not bool(dq[:, :5].any())
    out, dq, dk, dv = call(q, k, v, go, key_lengths=torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert not any(bool(t.any()) for t in (out, dq, dk, dv))
    out, dq, dk, dv = call(q, k[:, :0], v[:, :0], go)
    assert not bool(out.any()) and not bool(dq.any()) and dk.shape == (2, 0, 1, 16)
    out, dq, dk, dv = call(q[:, :0], k, v, go[:, :0])
    assert out.shape == (2, 0, 2, 16) and not bool(dk.any()) and not bool(dv.any())
    out, dq, dk, dv = call(q[:0], k[:0], v[:0], go[:0])
    assert out.shape == (0, 9, 2, 16) and dk.shape == (0, 4, 1, 16)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_what_is_not_seen_does_not_reach_a_result(dtype, bad):
    """Keys past key_lengths, later tokens and other sequences hold NaN and infinities; the
    results of those that do not see them are bit for bit those without."""
    # padding
    q, k, v, go = make(dtype, 2, 50, 90, 4, 2, 48)
    lengths = torch.tensor([37, 70], device="cuda")
    want = call(q, k, v, go, key_lengths=lengths)
    k2, v2 = k.clone(), v.clone()
    for b, n in enumerate((37, 70)):
        k2[b, n:], v2[b, n:] = bad, bad
    for x, w in zip(call(q, k2, v2, go, key_lengths=lengths), want):
        assert torch.equal(x, w)
    # the token at 60 of 100: earlier queries, and the keys behind it, do not meet it
    q, k, v, go = make(dtype, 1, 100, 100, 2, 2, 64)
    want = call(q, k, v, go, causal=True)
    k2, v2 = k.clone(), v.clone()
    k2[:, 60], v2[:, 60] = bad, bad
    out, dq, dk, dv = call(q, k2, v2, go, causal=True)
    assert torch.equal(out[:, :60], want[0][:, :60]) and torch.equal(dq[:, :60], want[1][:, :60])
    assert not bool(torch.isfinite(out[:, 60:]).any()) or bad == -math.inf
    q2, go2 = q.clone(), go.clone()
    q2[:, 60], go2[:, 60] = bad, bad
    out, dq, dk, dv = call(q2, k, v, go2, causal=True)
    others = torch.arange(100, device="cuda") != 60
    assert torch.equal(out[:, others], want[0][:, others]) and torch.equal(dq[:, others], want[1][:, others])
    assert torch.equal(dk[:, 61:], want[2][:, 61:]) and torch.equal(dv[:, 61:], want[3][:, 61:])
    assert not bool(torch.isfinite(dk[:, :61]).any()) and not bool(torch.isfinite(dv[:, :61]).any())
    # another sequence
    offsets = torch.tensor([0, 30, 75, 100], device="cuda")
    want = call(q[0], k[0], v[0], go[0], offsets=offsets)
    dirty = [t[0].clone() for t in (q, k, v, go)]
    for t in dirty:
        t[30:75] = bad
    for x, w in zip(call(*dirty, offsets=offsets), want):
        assert torch.equal(x[:30], w[:30]) and torch.equal(x[75:], w[75:])


def test_an_infinite_value_stays_infinite_where_it_is_seen():
    q, k, v, go = make("f32", 1, 40, 40, 1, 1, 32)
    v[0, 20, 0, 3] = math.inf
    with torch.no_grad():
        out = attention(q, k, v, causal=True)
    assert bool((out[0, 20:, 0, 3] == math.inf).all()) and bool(torch.isfinite(out[0, :20]).all())
    assert bool(torch.isfinite(out[0, 20:, 0, 4:]).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_scores_of_minus_infinity(dtype):
    """Keys that score -inf weigh nothing, also where a whole part of a long axis is of them; a query
    whose keys all score -inf has no softmax."""
    b, sk = 1, 1100
    q, k, v, go = make(dtype, b, 3, sk, 2, 1, 32)
    q = q.abs()
    for first, last in ((0, 700), (300, 1100), (64, 128)):
        k2 = k.clone()
        k2[:, first:last] = -math.inf
        seen = visible(b, 3, sk)
        seen[:, :, first:last] = False
        with torch.no_grad():
            out = attention(q, k2, v)
        want, bounds = definition(q, k, v, go, seen, dtype)
        within(out, want[0], bounds[0], "out")
    with torch.no_grad():
        assert bool(torch.isnan(attention(q, torch.full_like(k, -math.inf), v)).all())
        some = attention(q, torch.full_like(k, -math.inf), v, key_lengths=torch.tensor([0], device="cuda"))
        assert not bool(some.any())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("b,sq,sk,h,hk,d,causal", [(1, 2, 4100, 4, 1, 64, True), (3, 1, 2050, 8, 8, 128, False),
                                                   (1, 1500, 70, 8, 2, 40, False), (1, 1300, 1300, 2, 1, 96, True)])
def test_few_rows_over_a_long_axis(dtype, b, sq, sk, h, hk, d, causal):
    q, k, v, go = make(dtype, b, sq, sk, h, hk, d)
    compare(dtype, q, k, v, go, visible(b, sq, sk, causal), causal=causal)
    lengths = [sk // 3 + 7, 0, sk][:b]
    compare(dtype, q, k, v, go, visible(b, sq, sk, causal, lengths), causal=causal,
            key_lengths=torch.tensor(lengths, device="cuda"))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_strides_orders_and_alignment(dtype):
    b, s, h, hk, d = 2, 75, 4, 2, 40
    q, k, v, go = make(dtype, b, s, s, h, hk, d)
    want = call(q, k, v, go, causal=True)

    def check(*ts):
        for x, w in zip(call(*ts, causal=True), want):
            assert torch.equal(x, w)

    fused = torch.cat([t.reshape(b, s, -1) for t in (q, k, v)], 2)
    check(*(t.unflatten(-1, (-1, d)) for t in fused.split([h * d, hk * d, hk * d], 2)), go)
    head_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, go)]
    check(*head_first)
    token_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, go)]
    check(*token_first)
    odd = []
    for t in (q, k, v, go):  # one element off any alignment, rows of 41
        buf = torch.full((t.numel() // d * (d + 1) + 1,), math.nan, dtype=t.dtype, device="cuda")
        view = buf[1:].view(b, s, t.shape[2], d + 1)[..., :d]
        view.copy_(t)
        odd.append(view)
    check(*odd)
    check(*(t.transpose(-1, -2).contiguous().transpose(-1, -2) for t in (q, k, v, go)))  # width is not last
    # a gradient that is one value for all
    ones = call(q, k, v, torch.ones_like(go), causal=True)
    for x, w in zip(call(q, k, v, torch.ones((), dtype=go.dtype, device="cuda").expand(go.shape), causal=True), ones):
        assert torch.equal(x, w)


def test_a_negated_view_is_read_as_its_values():
    q, k, v, go = make("f32", 1, 20, 20, 2, 1, 16)
    want = call(-q, k, -v, go)
    neg = lambda t: torch.complex(torch.zeros_like(t), t).conj().imag  # noqa: E731
    assert neg(q).is_neg()
    for x, w in zip(call(neg(q), k, neg(v), go), want):
        assert torch.equal(x, w)


def test_shared_and_broadcast_operands():
    """Keys expanded to all sequences sum their gradients, as autograd's expand does."""
    q, k, v, go = make("f32", 3, 33, 50, 4, 2, 24)
    k1, v1 = k[:1].clone().requires_grad_(True), v[:1].clone().requires_grad_(True)
    out = attention(q, k1.expand(3, -1, -1, -1), v1.expand(3, -1, -1, -1))
    gk, gv = torch.autograd.grad(out, (k1, v1), grad_outputs=go)
    _, _, dk, dv = call(q, k[:1].expand(3, -1, -1, -1).contiguous(), v[:1].expand(3, -1, -1, -1).contiguous(), go)
    assert torch.equal(gk, dk.sum(0, keepdim=True)) and torch.equal(gv, dv.sum(0, keepdim=True))
    # one tensor as all three operands
    x = q.detach().requires_grad_(True)
    got, = torch.autograd.grad(attention(x, x, x, causal=True), (x,), grad_outputs=go)
    _, a, b, c = call(q, q, q, go, causal=True)
    assert torch.allclose(got, a + b + c, rtol=0, atol=4 * F * float((a.abs() + b.abs() + c.abs()).max()))


def test_only_some_gradients_are_wanted():
    q, k, v, go = make("bf16", 2, 40, 40, 4, 2, 32)
    _, dq, dk, dv = call(q, k, v, go)
    want = {"q": dq, "k": dk, "v": dv}
    for names in ("q", "k", "v", "qk", "kv", "qv"):
        ts = {n: t.detach().requires_grad_(n in names) for n, t in zip("qkv", (q, k, v))}
        attention(ts["q"], ts["k"], ts["v"]).backward(go)
        for n in "qkv":
            assert (ts[n].grad is None) == (n not in names)
            assert n not in names or torch.equal(ts[n].grad, want[n])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_calls_repeat_bit_for_bit(dtype):
    q, k, v, go = make(dtype, 2, 400, 400, 8, 2, 64)
    a, b = (call(q, k, v, go, causal=True) for _ in range(2))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_half_precision_gradients_of_small_and_large_scale():
    """Row gradients from 2^-20 to 2^10 keep a gradient's precision in dQ row by row, and large
    losses do not overflow on the way."""
    q, k, v, go = make("f16", 1, 96, 200, 2, 2, 64)
    go = go * torch.exp2(torch.linspace(-12, 9, 96, device="cuda"))[None, :, None, None].half()
    compare("f16", q, k, v, go, visible(1, 96, 200))
    q, k, v, go = make("f16", 1, 64, 64, 2, 2, 64)
    go = go * 4096.0
    compare("f16", q * 0.25, k * 0.25, v * 0.03125, go, visible(1, 64, 64, True), causal=True)


def test_gradients_agree_with_differences():
    """The derivative along a direction against a difference quotient of the operator itself.  The
    quotient's truncation is that of the definition's own, its rounding 2 sum |dO| eo / 2 h."""
    q, k, v, go = make("f32", 2, 23, 31, 4, 2, 24, seed=5)
    seen = visible(2, 23, 31, True)
    grads = call(q, k, v, go, causal=True)[1:]
    want, bounds = definition(q, k, v, go, seen, "f32")
    h = 2.0 ** -7
    g = torch.Generator(device="cuda").manual_seed(3)
    for which in range(3):
        step = torch.sign(torch.randn((q, k, v)[which].shape, device="cuda", generator=g)) * h
        ends, exact = [], []
        for s in (1, -1):
            ts = [t.clone() for t in (q, k, v)]
            ts[which] = ts[which] + s * step
            with torch.no_grad():
                ends.append(float((attention(*ts, causal=True).double() * go.double()).sum()))
            exact.append(float((definition(*ts, go, seen, "f32")[0][0] * go.double()).sum()))
        quotient, true_quotient = ends[0] - ends[1], exact[0] - exact[1]
        slope = float((grads[which].double() * 2 * step.double()).sum())
        true_slope = float((want[1 + which] * 2 * step.double()).sum())
        rounding = 2 * float((go.double().abs() * bounds[0]).sum()) * 1.25
        of_slope = float((bounds[1 + which] * 2 * h).sum())
        assert abs(quotient - slope) <= abs(true_quotient - true_slope) + rounding + of_slope


def test_a_captured_step_follows_its_inputs():
    q, k, v, go = make("bf16", 2, 130, 130, 4, 2, 64)
    lengths = torch.tensor([130, 77], dtype=torch.int32, device="cuda")
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]

    def step():
        out = attention(*leaves, causal=True, key_lengths=lengths)
        return (out,) + torch.autograd.grad(out, leaves, grad_outputs=go)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed, n in ((1, [130, 77]), (2, [5, 130]), (3, [0, 64])):
        fresh = make("bf16", 2, 130, 130, 4, 2, 64, seed=seed)
        with torch.no_grad():
            for t, x in zip(leaves + [go], fresh):
                t.copy_(x)
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for x, w in zip(got, call(*fresh, causal=True, key_lengths=lengths)):
            assert torch.equal(x.detach(), w)


def test_two_streams_at_once():
    a, b = make("bf16", 1, 600, 600, 8, 2, 64, seed=1), make("f16", 1, 500, 700, 6, 3, 80, seed=2)
    want = [call(*a, causal=True), call(*b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for s, ts, kw in zip(streams, (a, b), ({"causal": True}, {})):
            with torch.cuda.stream(s):
                got.append(call(*ts, **kw))
        torch.cuda.synchronize()
        for x, w in zip(got, want):
            assert all(torch.equal(i, j) for i, j in zip(x, w))


def test_far_rows_of_a_long_buffer():
    """Offsets past 2^31 elements: keys of the last of many sequences of one long cache."""
    from_end = 40
    big = torch.zeros((1 << 31) + (1 << 20), dtype=torch.bfloat16, device="cuda")
    rows = big.numel() // 128
    cache = big[:rows * 128].view(1, rows, 1, 128)
    q, k, v, go = make("bf16", 1, 3, from_end, 2, 1, 128)
    cache[:, rows - from_end:] = k
    far = cache[:, rows - from_end:]
    assert (far.data_ptr() - big.data_ptr()) // 2 > 1 << 31
    strided = torch.as_strided(big, (2, from_end, 1, 128), ((rows - from_end) * 128, 128, 128, 1))
    q2, v2 = q.expand(2, -1, -1, -1), v.expand(2, -1, -1, -1)
    with torch.no_grad():
        assert torch.equal(attention(q, far, v), attention(q, k, v))
        assert torch.equal(attention(q2, strided, v2)[1], attention(q, k, v)[0])


def test_autograd_is_told():
    q, k, v, go = (t.requires_grad_(i < 3) for i, t in enumerate(make("f32", 1, 8, 8, 2, 1, 16)))
    out = attention(q, k, v)
    grads = torch.autograd.grad(out, (q,), grad_outputs=go, retain_graph=True)
    assert torch.equal(grads[0], torch.autograd.grad(out, (q,), grad_outputs=go, retain_graph=True)[0])
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(out, (q,), grad_outputs=go, create_graph=True)
    out = attention(q, k, v)
    with torch.no_grad():
        k.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.backward(go)
    with pytest.raises(NotImplementedError, match="tangent"):
        import torch.autograd.forward_ad as fwd

        with fwd.dual_level():
            attention(fwd.make_dual(q.detach(), go), k, v)
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t.shape) or t, lambda t: t):
        attention(q, k, v)
    assert q.shape in seen and k.shape in seen


def test_refusals_on_the_device():
    q, k, v, go = make("bf16", 2, 8, 8, 4, 2, 16)
    lengths = torch.ones(2, dtype=torch.int32, device="cuda")
    bad = [((q, k.float(), v), {}), ((q, k, v[:, :4]), {}), ((q, k[..., :8], v[..., :8]), {}), ((q[:1], k, v), {}),
           ((q[:, :, :3], k, v), {}), ((q[0], k[0], v[0]), {}), ((q, k, v), {"offsets": lengths}),
           ((q, k, v), {"key_lengths": lengths[:1]}), ((q, k, v), {"key_lengths": lengths.float()}),
           ((q, k, v), {"key_lengths": lengths[None]}), ((q, k, v), {"key_lengths": lengths.cpu()}),
           ((q, k.cpu(), v), {}), ((q.double(), k.double(), v.double()), {}), ((q, k, v), {"scale": -1.0}),
           ((q, k, v), {"scale": math.inf}), ((q, k, v), {"scale": math.nan}),
           ((q[0], k[0], v[0]), {"offsets": lengths, "key_lengths": lengths}),
           ((q[0], k[0], v[0]), {"offsets": lengths[:0]}), ((q[0, :4], k[0], v[0]), {"offsets": lengths})]
    wide = torch.zeros(1, 4, 1, 129, dtype=torch.bfloat16, device="cuda")
    bad += [((wide, wide, wide), {}), ((wide[..., :0], wide[..., :0], wide[..., :0]), {}),
            ((q[:, :, :0], k, v), {}), ((q, k[:, :, :0], v[:, :, :0]), {})]
    for args, kw in bad:
        with pytest.raises(ValueError):
            attention(*args, **kw)
    with pytest.raises(TypeError):
        attention(q, k, None)
    with pytest.raises(TypeError):
        attention(q, k, v, key_lengths=[1, 2])
