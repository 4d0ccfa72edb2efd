"""Clipping refuses tensors whose memory it would write twice, or read after writing, before
anything is written; strided views that only interleave are taken."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def refused(call, *watch):
    before = [t.clone() for t in watch]
    with pytest.raises(ValueError, match="share no memory|overlap"):
        call()
    torch.cuda.synchronize()
    for t, b in zip(watch, before):
        assert torch.equal(t, b), "written before the refusal"


def test_expanded_gradients_and_outputs():
    from gefen_amd import clip_gradients

    a, x = torch.ones(50, device="cuda"), torch.ones(1, 4, device="cuda")
    refused(lambda: clip_gradients([a, x.expand(3, 4)], 0.1), a, x)
    refused(lambda: clip_gradients([a, torch.ones(3, 4, device="cuda")], 0.1, out=[torch.zeros_like(a), x.expand(3, 4)]),
            a, x)


def test_windows_that_overlap():
    from gefen_amd import clip_gradients

    a, x = torch.ones(50, device="cuda"), torch.ones(40, device="cuda")
    refused(lambda: clip_gradients([a, x.unfold(0, 8, 4)], 0.1), a, x)
    refused(lambda: clip_gradients([a, x.as_strided((3, 4), (5, 5))], 0.1), a, x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_tensors_of_the_same_memory(dtype):
    from gefen_amd import clip_gradients

    a = torch.ones(50, device="cuda")
    x = torch.ones(6, 8, device="cuda", dtype=dtype)
    refused(lambda: clip_gradients([a, x, x[:, ::2]], 0.1), a, x)
    refused(lambda: clip_gradients([a, x[:, ::2], x[:, 4:]], 0.1), a, x)
    refused(lambda: clip_gradients([a, x[:, ::2], x[:, ::2]], 0.1), a, x)
    refused(lambda: clip_gradients([a, x[2:], x.t()], 0.1), a, x)
    g = [torch.ones(6, 8, device="cuda"), torch.ones(6, 4, device="cuda")]
    refused(lambda: clip_gradients(g, 0.1, out=[x, x[:, ::2]]), x, *g)
    refused(lambda: clip_gradients([x[:, ::2]], 0.1, out=[x[:, 1:5]]), x)
    refused(lambda: clip_gradients([x[::2]], 0.1, out=[x[:3]]), x)


def test_views_that_only_interleave():
    from gefen_amd import clip_gradients

    x = torch.randn(64, 96, device="cuda")
    views = [x[:, :32], x[:, 32:64], x[:, 64::2], x[::2, 65::2], x[1::2, 65::2]]
    assert sum(v.numel() for v in views) == x.numel()
    want, norm = x.clone(), float(x.double().norm())
    total = clip_gradients(views, 1.0)
    assert abs(float(total) - norm) <= 2.0 ** -23 * norm
    want = want.double() / (norm + 1e-6)
    assert bool(((x.double() - want).abs() <= 2.0 ** -21 * want.abs()).all())
    a, b = torch.randn(7, 10, device="cuda").unbind(1)[3:5]
    big = torch.zeros(7, 4, device="cuda")
    clip_gradients([a, b], 1e6, out=[big[:, 1], big[:, 3]])
    assert torch.equal(big[:, 1], a) and torch.equal(big[:, 3], b) and bool((big[:, ::2] == 0).all())
    # one strided tensor into itself is in place
    y = torch.ones(8, 8, device="cuda")
    clip_gradients([y[:, ::2]], 1.0, out=[y[:, ::2]])
    assert bool((y[:, 1::2] == 1).all()) and bool((y[:, ::2] < 0.2).all())


def test_a_total_norm_inside_what_is_written():
    from gefen_amd import clip_gradients

    g = torch.full((20,), 4.0, device="cuda")
    refused(lambda: clip_gradients([g], 1.0, total_norm=g[3]), g)


def elements(t):
    """The positions of a tensor's elements in its memory."""
    at = torch.zeros((), dtype=torch.int64)
    for size, stride in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(size) * stride
    return (at + t.storage_offset()).reshape(-1).tolist()


def test_any_strides_are_told_apart():
    """Random views of one buffer: refused exactly where two elements, one of them written,
    share memory."""
    import random

    from gefen_amd import clip_gradients

    rng = random.Random(0)
    x = torch.ones(600, device="cuda")
    counts = {True: 0, False: 0}

    def view():
        shape = [rng.randint(1, 5) for _ in range(rng.randint(1, 3))]
        stride = [rng.choice([1, 2, 3, 4, 5, 8, 12, 16, 24, 48, 50]) for _ in shape]
        if rng.random() < 0.1:
            stride[0] = 0
        return x.as_strided(shape, stride, rng.randint(0, 60))

    for k in range(600):
        a, b = view(), view()
        if k % 3 == 2:  # a is read, b written
            b = x.as_strided(a.shape, b.stride()[:1] * a.dim() if a.dim() > b.dim() else b.stride()[:a.dim()],
                             b.storage_offset())
            same = elements(a) == elements(b)
            bad = len(set(elements(b))) < b.numel() or (bool(set(elements(a)) & set(elements(b))) and not same)
            if same and a.stride() != b.stride():
                continue  # one memory in one order, by other strides of single elements: either is right
            call = lambda: clip_gradients([a], 1e6, out=[b])
        else:
            every = elements(a) + elements(b)
            bad = len(set(every)) < len(every)
            call = lambda: clip_gradients([a, b], 1e6)
        counts[bad] += 1
        if bad:
            with pytest.raises(ValueError, match="share no memory|overlap"):
                call()
        else:
            call()
    assert min(counts.values()) > 100, counts


def test_an_expanded_gradient_beside_its_output():
    from gefen_amd import clip_gradients

    x = torch.zeros(6, 5, device="cuda")
    x[:, 0] = torch.arange(6.0)
    clip_gradients([x[:, :1].expand(6, 4)], 1e6, out=[x[:, 1:]])
    assert torch.equal(x, torch.arange(6.0, device="cuda")[:, None].expand(6, 5))
