"""Autograd is told of the tensors that clipping writes."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_clipping_counts_as_an_in_place_write():
    from gefen_amd import clip_grad_norm_, clip_gradients

    g = [torch.ones(5, 7, device="cuda"), torch.ones(9, 8, device="cuda")[:, ::2]]
    out = [torch.empty_like(t) for t in g]
    v = [t._version for t in g + out]
    clip_gradients(g, 1.0, out=out)
    assert [t._version for t in g] == v[:2] and all(t._version > u for t, u in zip(out, v[2:]))
    clip_gradients(g, 1.0)
    clip_gradients(g[:1], 1.0, total_norm=torch.tensor(4.0, device="cuda"))
    assert all(t._version > u for t, u in zip(g, v))
    p = torch.zeros(5, device="cuda", requires_grad=True)
    p.grad = torch.ones(5, device="cuda")
    u = p.grad._version
    clip_grad_norm_([p], 1e6)  # within the bound: as torch's, which multiplies by one
    assert p.grad._version > u


def test_a_saved_gradient_that_is_clipped_is_noticed():
    from gefen_amd import clip_gradients

    x = torch.randn(100, device="cuda", requires_grad=True)
    g, = torch.autograd.grad((x ** 3).sum(), x, create_graph=True)
    penalty = (g * g).sum()
    clip_gradients([g], 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        penalty.backward()
