"""The training operators together: the example's loop learns, its clipped gradients are
those of a plain computation, and the step that follows takes them."""

import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))


def test_the_example_learns():
    from train_step import train

    losses, norms = train(steps=60, vocab=1009, width=128, rows=8, length=60, report=0)
    assert len(losses) == 60 and all(x == x and x > 0 for x in losses + norms)
    assert sum(losses[-5:]) < 0.6 * sum(losses[:5])


def test_clipped_gradients_are_the_plain_ones():
    """One backward pass and clip of the example's model against torch's cross entropy and
    clip in float32.  The head's gradient is off by its terms' roundings (2^-8 of each at
    most, of independent sign) and its own; the layers below take hidden's rounded gradient
    through bfloat16 products: a relative 2^-5 of a tensor's norm covers either."""
    from train_step import Model, batch

    from gefen_amd import clip_grad_norm_

    torch.manual_seed(0)
    model = Model(1009, 128).bfloat16().cuda()
    tokens, targets = batch(torch.Generator().manual_seed(2), 1009, 8, 60)
    model.loss(tokens, targets).backward()
    plain = Model(1009, 128).cuda()
    plain.load_state_dict({k: v.float() for k, v in model.state_dict().items()})
    logits = plain(tokens) @ plain.head.weight.t()
    torch.nn.functional.cross_entropy(logits.reshape(-1, 1009), targets.reshape(-1)).backward()
    bound = 0.5 * float(torch.nn.utils.clip_grad_norm_(plain.parameters(), float("inf")))
    want_norm = torch.nn.utils.clip_grad_norm_(plain.parameters(), bound)
    norm = clip_grad_norm_(model.parameters(), bound)
    got = [p.grad.float() for p in model.parameters()]
    assert abs(float(norm) - float(want_norm)) <= 2.0 ** -5 * float(want_norm)
    for g, p in zip(got, plain.parameters()):
        assert float((g - p.grad).norm()) <= 2.0 ** -5 * float(p.grad.norm())
