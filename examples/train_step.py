"""One training loop with what this package has for a step around the model:

    loss = linear_cross_entropy(hidden, head, targets)   # no logits are kept
    loss.backward()
    norm = clip_grad_norm_(parameters, max_norm)
    optimizer.step()                                     # Gefen

on a small bfloat16 language model that learns a made-up sequence rule.

    python examples/train_step.py [--steps 60] [--vocab 5003] [--width 256]
"""

import argparse
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import torch  # noqa: E402

from gefen import Gefen  # noqa: E402
from gefen_amd import clip_grad_norm_, linear_cross_entropy  # noqa: E402


class Model(torch.nn.Module):
    """Embedding, one gated layer, output matrix."""

    def __init__(self, vocab, width):
        super().__init__()
        self.embed = torch.nn.Embedding(vocab, width)
        self.gate = torch.nn.Linear(width, 2 * width, bias=False)
        self.up = torch.nn.Linear(width, 2 * width, bias=False)
        self.down = torch.nn.Linear(2 * width, width, bias=False)
        self.head = torch.nn.Linear(width, vocab, bias=False)

    def forward(self, tokens):
        x = self.embed(tokens)
        return x + self.down(torch.nn.functional.silu(self.gate(x)) * self.up(x))

    def loss(self, tokens, targets):
        return linear_cross_entropy(self(tokens), self.head.weight, targets)


def batch(generator, vocab, rows, length):
    """Sequences in which the next token is three times the last one plus one, modulo 97,
    except for one in eight, which is any; a third of each sequence is a prompt that has no
    loss."""
    t = torch.empty(rows, length + 1, dtype=torch.int64)
    t[:, 0] = torch.randint(0, vocab, (rows,), generator=generator)
    for i in range(1, length + 1):
        noise = torch.randint(0, vocab, (rows,), generator=generator)
        rule = (3 * t[:, i - 1] + 1) % 97 % vocab
        t[:, i] = torch.where(torch.rand(rows, generator=generator) < 0.125, noise, rule)
    targets = t[:, 1:].clone()
    targets[:, :length // 3] = -100
    return t[:, :-1].cuda(), targets.cuda()


def train(steps=60, vocab=5003, width=256, rows=16, length=96, lr=3e-3, max_norm=1.0, report=10):
    """Returns the losses and the gradient norms of all steps."""
    torch.manual_seed(0)
    generator = torch.Generator().manual_seed(1)
    model = Model(vocab, width).bfloat16().cuda()
    optimizer = Gefen(model.named_parameters(), lr=lr)
    losses, norms = [], []
    for step in range(steps):
        tokens, targets = batch(generator, vocab, rows, length)
        loss = model.loss(tokens, targets)
        loss.backward()
        norm = clip_grad_norm_(model.parameters(), max_norm)
        optimizer.step()
        optimizer.zero_grad()
        losses.append(loss.detach())
        norms.append(norm)
        if report and step % report == 0:
            print("step {:4d}  loss {:.4f}  gradient norm {:.4f}".format(step, loss.item(), norm.item()), flush=True)
    return torch.stack(losses).tolist(), torch.stack(norms).tolist()


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--vocab", type=int, default=5003)
    ap.add_argument("--width", type=int, default=256)
    args = ap.parse_args()
    losses, _ = train(args.steps, args.vocab, args.width)
    print("loss {:.4f} -> {:.4f} in {} steps".format(losses[0], losses[-1], len(losses)))
