"""Forward-mode tangents are refused, not dropped."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_tangents_are_refused():
    import torch.autograd.forward_ad as fwd

    from gefen_amd import clip_gradients, gradient_norm, linear_cross_entropy

    h, w = torch.randn(5, 16, device="cuda"), torch.randn(9, 16, device="cuda")
    y = torch.zeros(5, dtype=torch.int64, device="cuda")
    with fwd.dual_level():
        dual = fwd.make_dual(h, torch.ones_like(h))
        for call in (lambda: linear_cross_entropy(dual, w, y),
                     lambda: linear_cross_entropy(h, fwd.make_dual(w, torch.ones_like(w)), y),
                     lambda: linear_cross_entropy(dual, w.clone().requires_grad_(True), y),
                     lambda: gradient_norm([h, dual]), lambda: clip_gradients([h.clone(), dual], 1.0)):
            with pytest.raises(NotImplementedError, match="forward"):
                call()
        # no tangent: as outside of the level
        assert torch.equal(linear_cross_entropy(h, w, y), linear_cross_entropy(h, w.clone(), y))
