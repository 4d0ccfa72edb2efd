"""gradient_norm, clip_gradients and clip_grad_norm_ against float64, and what they refuse.

The norm's sums are float64 of exact squares; it is rounded to float32 once, and the
root's and the sum's own errors are far below: within 2^-23 of the float64 result.  The
coefficient adds two float32 roundings, and the product one in float32 and one to the
dtype (half its spacing at 1: 2^-24, 2^-11, 2^-8)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def grads_of(sizes, dtypes, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale * 2.0 ** (i % 5 - 4)).to(DT[dtypes[i % len(dtypes)]]).cuda()
            for i, n in enumerate(sizes)]


def norm64(grads, kind=2.0):
    flat = [g.double().abs().reshape(-1) for g in grads if g.numel()]
    if not flat:
        return 0.0
    if kind == math.inf:
        return max(float(f.max()) for f in flat)
    if kind == 1.0:
        return math.fsum(float(f.sum()) for f in flat)
    return math.sqrt(math.fsum(float(f.square().sum()) for f in flat))


def check_scaled(before, after, norm, bound):
    c = min(1.0, bound / (norm + 1e-6))
    for b, a in zip(before, after):
        want = b.double() * c
        err = (a.double() - want).abs()
        assert bool((err <= want.abs() * (U[a.dtype] + 5 * 2.0 ** -24) + TINY[a.dtype]).all()), (b.shape, a.dtype)


SETS = [[1], [0, 5, 0], [16384], [16385, 1], [3, 70000, 16383, 8, 0, 1], [257] * 300, [1 << 20, 777, 1 << 18, 5],
        [5000017]]


@pytest.mark.parametrize("dtypes", [["f32"], ["bf16"], ["f16"], ["bf16", "f32", "f16"]])
@pytest.mark.parametrize("sizes", SETS)
def test_norms_and_clipping_match_float64(sizes, dtypes):
    from gefen_amd import clip_gradients, gradient_norm

    grads = grads_of(sizes, dtypes)
    for kind in (1.0, 2.0, math.inf):
        want = norm64(grads, kind)
        got = gradient_norm(grads, kind)
        assert got.dtype == torch.float32 and got.dim() == 0 and got.is_cuda
        assert abs(float(got) - want) <= 2.0 ** -23 * want, kind
        for bound in (0.3 * want, 3.0 * want + 1.0):
            mine = [g.clone() for g in grads]
            total = clip_gradients(mine, bound, kind)
            assert torch.equal(total, got)
            check_scaled(grads, mine, want, bound)
            if bound > want:
                assert all(torch.equal(a, b) for a, b in zip(grads, mine))


@pytest.mark.parametrize("src,dst", [("f32", "bf16"), ("f32", "f16"), ("bf16", "f32"), ("f16", "bf16"), ("bf16", "bf16")])
def test_into_other_buffers(src, dst):
    from gefen_amd import clip_gradients

    grads = grads_of([7, 40000, 0, 16384, 129], [src], seed=1, scale=0.1)
    keep = [g.clone() for g in grads]
    for bound in (0.5, 1e6):
        out = [torch.full_like(g, 9.0, dtype=DT[dst]) for g in grads]
        total = clip_gradients(grads, bound, out=out)
        want = norm64(grads)
        assert abs(float(total) - want) <= 2.0 ** -23 * want
        check_scaled(grads, out, want, bound)
        assert all(torch.equal(a, b) for a, b in zip(grads, keep))


def test_any_layout_and_alignment():
    """Views that start off any alignment, transposed ones, columns, rows of a wider matrix."""
    from gefen_amd import clip_gradients, gradient_norm

    base = torch.randn(400, 300, device="cuda").bfloat16()
    flat = torch.randn(50001, device="cuda")
    views = [base[:50].t(), base[100:200, 7:205], flat[3:40002], base[210], base[300:, 5], flat[45000:45001]]
    before = [v.clone() for v in views]
    rest = flat[40002:45000].clone()
    edge = base[100:200, :7].clone()
    want = norm64(before)
    assert abs(float(gradient_norm(views)) - want) <= 2.0 ** -23 * want
    out = [torch.empty(v.shape, device="cuda").t().contiguous().t() if v.dim() == 2 else torch.empty_like(v) for v in views]
    clip_gradients(views, 1.0, out=out)
    check_scaled(before, out, want, 1.0)
    clip_gradients(views, 1.0)
    check_scaled(before, views, want, 1.0)
    assert torch.equal(flat[40002:45000], rest) and torch.equal(base[100:200, :7], edge)


def test_range_of_float32():
    """Squares that would overflow or vanish in float32."""
    from gefen_amd import clip_gradients, gradient_norm

    big = [torch.full((1000,), 1e30, device="cuda")]
    assert abs(float(gradient_norm(big)) / (1e30 * math.sqrt(1000)) - 1) < 2.0 ** -22
    small = [torch.full((1000,), 1e-30, device="cuda")]
    assert abs(float(gradient_norm(small)) / (1e-30 * math.sqrt(1000)) - 1) < 2.0 ** -22
    clip_gradients(big, 2.0)
    assert abs(norm64(big) - 2.0) < 1e-5


def test_non_finite_gradients():
    from gefen_amd import clip_grad_norm_, clip_gradients, gradient_norm

    for kind in (1.0, 2.0, math.inf):
        g = [torch.ones(5000, device="cuda"), torch.ones(7, device="cuda").bfloat16()]
        g[1][3] = float("nan")
        assert bool(torch.isnan(gradient_norm(g, kind)))
        clip_gradients(g, 1.0, kind)
        assert all(bool(torch.isnan(t).all()) for t in g)
        g = [torch.ones(5000, device="cuda"), torch.ones(7, device="cuda").bfloat16()]
        g[0][11] = -float("inf")
        assert float(clip_gradients(g, 1.0, kind)) == math.inf
        assert bool(torch.isnan(g[0][11])) and float(g[0][0]) == 0.0 and float(g[1][0]) == 0.0
    p = torch.zeros(10, device="cuda", requires_grad=True)
    p.grad = torch.full((10,), float("nan"), device="cuda")
    p.grad[0] = 1.0
    with pytest.raises(RuntimeError, match="non-finite"):
        clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
    assert float(p.grad[0]) == 1.0


def test_clip_grad_norm_as_torch_has_it():
    from gefen_amd import clip_grad_norm_

    g = torch.Generator().manual_seed(2)
    ps = [torch.zeros(s, device="cuda", requires_grad=True) for s in [(30, 40), (7,), (1,), (500, 300)]]
    qs = [p.detach().clone().requires_grad_(True) for p in ps]
    for p, q in zip(ps[:-1], qs[:-1]):
        p.grad = torch.randn(p.shape, generator=g).cuda()
        q.grad = p.grad.clone()
    a = clip_grad_norm_(iter(ps), 1.5)
    b = torch.nn.utils.clip_grad_norm_(qs, 1.5)
    assert abs(float(a) - float(b)) <= 1e-6 * float(b)
    for p, q in zip(ps[:-1], qs[:-1]):
        assert bool(((p.grad - q.grad).abs() <= 1e-6 * q.grad.abs()).all())
    assert ps[-1].grad is None
    assert float(clip_grad_norm_([], 1.0)) == 0.0 and float(clip_grad_norm_([ps[-1]], 1.0)) == 0.0
    assert float(clip_grad_norm_(ps[0], 100.0)) > 0.0


def test_a_shard_is_scaled_by_the_whole_norm():
    from gefen_amd import clip_gradients, gradient_norm

    shards = [grads_of([5000, 31], ["bf16"], seed=3), grads_of([5000, 31], ["bf16"], seed=4)]
    norms = [gradient_norm(s) for s in shards]
    whole = (norms[0].square() + norms[1].square()).sqrt()
    before = [[g.clone() for g in s] for s in shards]
    for s, b in zip(shards, before):
        assert clip_gradients(s, 1.0, total_norm=whole) is whole
        check_scaled(b, s, float(whole), 1.0)


def test_norms_repeat_bit_for_bit_on_any_stream():
    from gefen_amd import gradient_norm

    grads = grads_of([1 << 22, 333, 1 << 20], ["bf16", "f32"], seed=5)
    first = gradient_norm(grads)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = [gradient_norm(grads) for _ in range(5)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(first, a) for a in again)


def test_a_captured_clip_replays():
    from gefen_amd import clip_gradients

    src = grads_of([4000, 70001, 5], ["f32"], seed=6)
    out = [torch.zeros_like(g, dtype=torch.bfloat16) for g in src]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        clip_gradients(src, 1.0, out=out)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_gradients(src, 1.0, out=out)
    for k in range(4):
        for g, new in zip(src, grads_of([4000, 70001, 5], ["f32"], seed=10 + k)):
            g.copy_(new)
        want = [torch.zeros_like(o) for o in out]
        total = clip_gradients(src, 1.0, out=want)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, total) and all(torch.equal(a, b) for a, b in zip(out, want))


def test_more_than_2_32_elements():
    from gefen_amd import clip_gradients, gradient_norm

    n = (1 << 32) + 77
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g[0], g[(1 << 31) + 5], g[n - 1] = 3.0, 4.0, 12.0
    assert float(gradient_norm([g])) == 13.0
    clip_gradients([g], 6.5)
    assert [float(g[i]) for i in (0, (1 << 31) + 5, n - 1)] == [1.5, 2.0, 6.0]


def test_refusals():
    from gefen_amd import clip_grad_norm_, clip_gradients, gradient_norm

    g = torch.ones(8, device="cuda")
    with pytest.raises(TypeError):
        gradient_norm({"g": g})
    with pytest.raises(TypeError):
        gradient_norm([g, 1.0])
    with pytest.raises(ValueError, match="CUDA"):
        gradient_norm([g, g.cpu()])
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        gradient_norm([g.double()])
    with pytest.raises(ValueError, match="norm_type"):
        gradient_norm([g], 3.0)
    with pytest.raises(ValueError, match="max_norm"):
        clip_gradients([g], -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        clip_grad_norm_([g], float("nan"))
    with pytest.raises(ValueError, match="as many"):
        clip_gradients([g], 1.0, out=[])
    with pytest.raises(ValueError, match="shapes"):
        clip_gradients([g], 1.0, out=[torch.empty(9, device="cuda")])
    with pytest.raises(ValueError, match="share no memory"):
        clip_gradients([g, g], 1.0)
    with pytest.raises(ValueError, match="share no memory"):
        clip_gradients([g[:4]], 1.0, out=[g[2:6]])
    with pytest.raises(ValueError, match="0-d float32"):
        clip_gradients([g], 1.0, total_norm=torch.ones(1, device="cuda"))
    assert bool((g == 1).all())
