"""Views that stand for the negative of their memory."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_negated_views_have_their_values():
    """The imaginary part of a conjugate is a view that stands for the negative of its memory."""
    from gefen_amd import clip_gradients, linear_cross_entropy

    torch.manual_seed(4)

    def negated(x):
        t = torch.complex(torch.zeros_like(x), -x).conj().imag
        assert t.is_neg() and torch.equal(t, x)
        return t

    h, w = torch.randn(30, 16, device="cuda"), torch.randn(50, 16, device="cuda")
    y = torch.randint(0, 50, (30,), device="cuda")
    want = linear_cross_entropy(h, w, y)
    assert torch.equal(linear_cross_entropy(negated(h), w, y), want)
    assert torch.equal(linear_cross_entropy(h, negated(w), y), want)
    out = [torch.empty_like(h)]
    clip_gradients([negated(h)], 1e6, out=out)
    assert torch.equal(out[0], h)
    t = negated(h)
    clip_gradients([t], 1.0)
    expect = [h.clone()]
    clip_gradients(expect, 1.0)
    assert torch.equal(t, expect[0])
