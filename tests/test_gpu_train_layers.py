"""The layer operators together, as the example's decoder uses them: the loss and every
parameter's gradient against a float64 computation of the same model, and the loop runs."""

import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))


def plain_loss(model, params, tokens, offsets, targets, masks):
    """The model's loss from elementary operations on `params` (name -> float64 leaf)."""
    p = lambda name: params[name]  # noqa: E731
    norm = lambda s, w: s * torch.rsqrt(s.square().mean(-1, keepdim=True) + 1e-6) * w  # noqa: E731
    n = tokens.numel()
    of = torch.bucketize(torch.arange(n, device="cuda"), offsets[1:], right=True)
    i = torch.arange(n, device="cuda")
    seen = (of[:, None] == of[None]) & (i[None] <= i[:, None])
    s = p("embed.weight")[tokens] * masks[0]
    names = [f"layers.{k}.{w}" for k in range(len(model.layers)) for w in ("norm", "norm_gated")] + ["norm"]
    y = norm(s, p(names[0]))
    for k, layer in enumerate(model.layers):
        pre, h, d = f"layers.{k}.", layer.heads, layer.each
        q, key, v = (y @ p(pre + "qkv.weight").t()).unflatten(-1, (-1, d)).split([h, h // 2, h // 2], -2)
        key, v = key.repeat_interleave(2, 1), v.repeat_interleave(2, 1)
        outs = []
        for head in range(h):
            logits = (q[:, head] @ key[:, head].t() / d ** 0.5).masked_fill(~seen, -float("inf"))
            outs.append(torch.softmax(logits, 1) @ v[:, head])
        a = torch.cat(outs, -1) @ p(pre + "out.weight").t()
        s = s + a * masks[2 * k + 1]
        y = norm(s, p(names[2 * k + 1]))
        g = torch.nn.functional.silu(y @ p(pre + "gate.weight").t()) * (y @ p(pre + "up.weight").t())
        s = s + g @ p(pre + "down.weight").t() * masks[2 * k + 2]
        y = norm(s, p(names[2 * k + 2]))
    return torch.nn.functional.cross_entropy(y @ p("head.weight").t(), targets)


@pytest.mark.parametrize("dtype,share", [(torch.float32, 2.0 ** -12), (torch.bfloat16, 2.0 ** -4)])
def test_gradients_of_a_decoder(dtype, share):
    """Every intermediate is off by a few roundings u of its own size (float32 operands of the loss are
    taken in 22 bits), forward and backward pass through some 60 operations in a row, and a
    normalised stream keeps relative sizes: 60 * 4 u of a tensor's norm is 2^-16 in float32 (2^-14
    with the 22 bits) and, at 2^-8 with errors of independent sign, sqrt(60) 2^-8 = 2^-5 in
    bfloat16; twice to four times that is allowed."""
    from train_layers import Model, batch

    from gefen_amd import dropout

    torch.manual_seed(0)
    model = Model(503, 64, 2).to(dtype).cuda()
    tokens, offsets, targets = batch(torch.Generator().manual_seed(2), 503, 400)
    seed = torch.tensor(77, dtype=torch.int64, device="cuda")
    loss = model.loss(tokens, offsets, targets, seed)
    loss.backward()
    ones = torch.ones(tokens.numel(), 64, device="cuda")
    masks = [dropout(ones, model.p, 77, offset=k).double() for k in range(5)]
    params = {k: v.detach().double().requires_grad_(True) for k, v in model.named_parameters()}
    want = plain_loss(model, params, tokens, offsets, targets, masks)
    grads = dict(zip(params, torch.autograd.grad(want, list(params.values()))))
    assert abs(float(loss) - float(want)) <= share * abs(float(want))
    for name, v in model.named_parameters():
        assert float((v.grad.double() - grads[name]).norm()) <= share * float(grads[name].norm()), name


def test_the_example_runs():
    from train_layers import train

    losses, norms = train(steps=6, vocab=503, width=64, layers=1, tokens=300, report=0)
    assert len(losses) == len(norms) == 6 and all(x == x and 0 < x < float("inf") for x in losses + norms)
