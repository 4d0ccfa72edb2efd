"""A training loop of a small decoder whose layers run on this package's operators:

    y = rms_norm(s, w)                                            # of the residual stream s
    a = attention(q, k, v, causal=True, offsets=offsets)          # packed sequences
    y, s = rms_norm(out(a), w, residual=s, dropout=p, seed=seed)  # s + dropout(out(a)), and its norm
    loss = linear_cross_entropy(y, head, targets)
    loss.backward(); clip_grad_norm_(parameters, 1.0); optimizer.step()

on sequences of uneven length in one row of tokens, without padding.

    python examples/train_layers.py [--steps 40] [--vocab 5003] [--width 256] [--layers 2]
"""

import argparse
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import torch  # noqa: E402

from gefen import Gefen  # noqa: E402
from gefen_amd import attention, clip_grad_norm_, dropout, linear_cross_entropy, rms_norm  # noqa: E402


class Layer(torch.nn.Module):
    """Attention of `heads` heads over half as many key heads, and a gated layer."""

    def __init__(self, width, heads):
        super().__init__()
        self.heads, self.each = heads, width // heads
        self.qkv = torch.nn.Linear(width, 2 * width, bias=False)
        self.out = torch.nn.Linear(width, width, bias=False)
        self.gate = torch.nn.Linear(width, 2 * width, bias=False)
        self.up = torch.nn.Linear(width, 2 * width, bias=False)
        self.down = torch.nn.Linear(2 * width, width, bias=False)
        self.norm = torch.nn.Parameter(torch.ones(width))
        self.norm_gated = torch.nn.Parameter(torch.ones(width))

    def attend(self, y, offsets):
        q, k, v = self.qkv(y).unflatten(-1, (-1, self.each)).split([self.heads, self.heads // 2, self.heads // 2], -2)
        return self.out(attention(q, k, v, causal=True, offsets=offsets).flatten(-2))

    def gated(self, y):
        return self.down(torch.nn.functional.silu(self.gate(y)) * self.up(y))


class Model(torch.nn.Module):
    def __init__(self, vocab, width, layers, heads=4, p=0.1):
        super().__init__()
        self.p = p
        self.embed = torch.nn.Embedding(vocab, width)
        self.layers = torch.nn.ModuleList([Layer(width, heads) for _ in range(layers)])
        self.norm = torch.nn.Parameter(torch.ones(width))
        self.head = torch.nn.Linear(width, vocab, bias=False)

    def forward(self, tokens, offsets, seed):
        """The normed residual stream of packed tokens; each place of dropout has an offset of
        its own in the generator."""
        s = dropout(self.embed(tokens), self.p, seed)
        norms = [n for layer in self.layers for n in (layer.norm, layer.norm_gated)] + [self.norm]
        y = rms_norm(s, norms[0])
        for i, layer in enumerate(self.layers):
            for k, branch in enumerate((lambda y: layer.attend(y, offsets), layer.gated)):
                at = 2 * i + k + 1
                y, s = rms_norm(branch(y), norms[at], residual=s, dropout=self.p, seed=seed, offset=at)
        return y

    def loss(self, tokens, offsets, targets, seed):
        return linear_cross_entropy(self(tokens, offsets, seed), self.head.weight, targets)


def batch(generator, vocab, tokens):
    """Packed sequences of 1 to 200 tokens in which the next token repeats one of a few before
    it; their last positions have no target."""
    lengths = []
    while sum(lengths) < tokens:
        lengths.append(min(int(torch.randint(1, 201, (), generator=generator)), tokens - sum(lengths)))
    out, targets = [], []
    for n in lengths:
        t = torch.randint(0, vocab, (n + 1,), generator=generator)
        back = torch.randint(1, 4, (n + 1,), generator=generator)
        for i in range(1, n + 1):
            if i >= back[i] and back[i] < 3:
                t[i] = t[i - back[i]]
        out.append(t[:n])
        targets.append(torch.cat([t[1:n], torch.tensor([-100])]))
    offsets = torch.tensor([0] + lengths).cumsum(0).to(torch.int32)
    return torch.cat(out).cuda(), offsets.cuda(), torch.cat(targets).cuda()


def train(steps=40, vocab=5003, width=256, layers=2, tokens=1500, lr=2e-3, max_norm=1.0, report=10):
    """Returns the losses and the gradient norms of all steps."""
    torch.manual_seed(0)
    generator = torch.Generator().manual_seed(1)
    model = Model(vocab, width, layers).bfloat16().cuda()
    optimizer = Gefen(model.named_parameters(), lr=lr)
    seed = torch.tensor(0, dtype=torch.int64, device="cuda")  # counted up: another mask every step
    losses, norms = [], []
    for step in range(steps):
        tokens_, offsets, targets = batch(generator, vocab, tokens)
        loss = model.loss(tokens_, offsets, targets, seed)
        loss.backward()
        norm = clip_grad_norm_(model.parameters(), max_norm)
        optimizer.step()
        optimizer.zero_grad()
        seed += 1
        losses.append(loss.detach())
        norms.append(norm)
        if report and step % report == 0:
            print("step {:4d}  loss {:.4f}  gradient norm {:.4f}".format(step, loss.item(), norm.item()), flush=True)
    return torch.stack(losses).tolist(), torch.stack(norms).tolist()


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--vocab", type=int, default=5003)
    ap.add_argument("--width", type=int, default=256)
    ap.add_argument("--layers", type=int, default=2)
    args = ap.parse_args()
    losses, _ = train(args.steps, args.vocab, args.width, args.layers)
    print("loss {:.4f} -> {:.4f} in {} steps".format(losses[0], losses[-1], len(losses)))
