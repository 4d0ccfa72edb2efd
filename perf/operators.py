"""The operators of a training step beside the optimizer, as timed cases.

Two operators, four kinds of call, each through the public entry points:

* ``norm``: the global norm of a model's gradients;
* ``clip``: that norm, and the gradients scaled to a bound, in place or into other buffers;
* ``eval``: the loss of every position from hidden states and an output matrix, no gradient;
* ``train``: the mean loss and the gradients of the hidden states and of the output matrix.

With ``own`` false the same results come from elementary torch operations in 32 bits.
Models are those of bench.py's configurations, the tests' small ones, or of odd sizes
drawn from a seed.
"""

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6      # added to the norm that max_norm is divided by
ALIGN = 256     # elements between tensors of a flat buffer, as torch's allocator aligns them
IGNORE = -100   # target of a position that has no loss


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the norm of a small model's gradients, logged every step: all latency
        {"name": "norm small mlp f32", "kind": "norm", "net": "mlp", "dtype": "f32", "width": 96, "layers": 3,
         "vocab": 64},
        # the norm of an 8B model's gradients: the largest set
        {"name": "norm llama8b bf16", "kind": "norm", "net": "llama", "dtype": "bf16", "width": 4096, "layers": 32,
         "kv": 1024, "inter": 14336, "vocab": 128256},
        # every step of a float32 run whose gradients stay within the bound
        {"name": "clip gpt2 f32", "kind": "clip", "net": "gpt2", "dtype": "f32", "width": 768, "layers": 12,
         "vocab": 50257, "out": None, "max_norm": 1e4},
        # gradients accumulated over micro-batches in float32, clipped into the bf16 ones of the step
        {"name": "clip llama1.5b f32 into bf16", "kind": "clip", "net": "llama", "dtype": "f32", "width": 2048,
         "layers": 16, "kv": 512, "inter": 8192, "vocab": 128256, "out": "bf16", "max_norm": 1.0},
        # float16 gradients of odd sizes beside float32 ones of vectors, some of them empty
        {"name": "clip ragged f16", "kind": "clip", "net": "ragged", "dtype": "f16", "tensors": 120, "side": 900,
         "mix": 5, "out": "same", "max_norm": 0.5},
        # the loss of one position, as a scoring loop asks for it: one pass over the output matrix
        {"name": "eval one token bf16", "kind": "eval", "dtype": "bf16", "n": 1, "v": 128256, "d": 2048,
         "ignored": 0, "smoothing": 0.0},
        # a validation batch of odd length in float32
        {"name": "eval gpt2 f32", "kind": "eval", "dtype": "f32", "n": 777, "v": 50257, "d": 768,
         "ignored": 13, "smoothing": 0.0},
        # a test-sized model's step: all latency
        {"name": "train small bf16", "kind": "train", "dtype": "bf16", "n": 48, "v": 1000, "d": 96,
         "ignored": 5, "smoothing": 0.0, "scale": 1.0},
        # eight sequences of 1024 through the float32 GPT-2 head
        {"name": "train gpt2 f32", "kind": "train", "dtype": "f32", "n": 8192, "v": 50257, "d": 768,
         "ignored": 8, "smoothing": 0.0, "scale": 1.0},
        # one micro-batch of four of a fine-tuning run: prompts are masked, the gradient is scaled by 1/4
        {"name": "train llama1.5b bf16", "kind": "train", "dtype": "bf16", "n": 4096, "v": 128256, "d": 2048,
         "ignored": 1300, "smoothing": 0.0, "scale": 0.25},
        # float16 with a loss scale, label smoothing, and sizes that divide badly
        {"name": "train odd f16", "kind": "train", "dtype": "f16", "n": 1531, "v": 32003, "d": 1001,
         "ignored": 400, "smoothing": 0.1, "scale": 1024.0},
        # a batch of 8192 positions through the 8B head: the largest
        {"name": "train llama8b bf16", "kind": "train", "dtype": "bf16", "n": 8192, "v": 128256, "d": 4096,
         "ignored": 2, "smoothing": 0.0, "scale": 1.0},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed ones' ranges, at most as large as the largest of its kind."""
    kind = rng.choice(["norm", "clip", "eval", "train", "train"])
    case = {"kind": kind}
    if kind in ("norm", "clip"):
        net = rng.choice(["mlp", "gpt2", "llama", "ragged"])
        case.update(net=net, dtype=rng.choice(["f32", "bf16", "f16"]))
        if net == "mlp":
            case.update(width=_spread(rng, 3, 1500), layers=rng.randint(1, 8), vocab=_spread(rng, 2, 4000))
        elif net == "gpt2":
            case.update(width=64 * rng.randint(2, 12), layers=rng.randint(1, 12), vocab=_spread(rng, 500, 50257))
        elif net == "llama":
            width = 256 * rng.randint(1, 8)
            case.update(width=width, layers=rng.randint(1, 16), kv=width // 4, inter=128 * rng.randint(4, 64),
                        vocab=_spread(rng, 500, 128256))
        else:
            case.update(tensors=rng.randint(1, 400), side=_spread(rng, 5, 900), mix=rng.randint(0, 9999))
        if kind == "clip":
            # in place only within the bound: a pass leaves its gradients as the next one takes them
            out = rng.choice([None, "same", "bf16", "f32"])
            case.update(out=out, max_norm=1e6 if out is None else rng.choice([0.1, 1.0, 1e6]))
        return case
    case["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32"])
    while True:
        n, v, d = _spread(rng, 1, 8192), _spread(rng, 300, 151936), _spread(rng, 48, 4096)
        if rng.random() < 0.5:
            d = -(-d // 64) * 64
        if n * v * d <= (8192 * 128256 * 4096 if case["dtype"] != "f32" else 8192 * 50257 * 768):
            break
    part = rng.choice([0.0, 0.0, 0.1, 0.5, 0.9])
    case.update(n=n, v=v, d=d, ignored=min(n - 1, int(part * n)), smoothing=rng.choice([0.0, 0.0, 0.1]))
    if kind == "train":
        case["scale"] = 1024.0 if case["dtype"] == "f16" else rng.choice([1.0, 1.0, 0.25])
    return case


# ------------------------------------------------------------------ shapes
def _shapes(case):
    net, w = case["net"], case.get("width", 0)
    out = []
    if net == "mlp":
        out.append((w, case["vocab"]))
        for _ in range(case["layers"]):
            out += [(w, w), (w,)]
        out += [(case["vocab"], w), (case["vocab"],)]
    elif net == "gpt2":
        out = [(case["vocab"], w), (1024, w)]
        for _ in range(case["layers"]):
            out += [(w, 3 * w), (3 * w,), (w, w), (w, 4 * w), (4 * w, w), (w,), (w,), (w,), (w,)]
        out.append((w,))
    elif net == "llama":
        kv, inter = case["kv"], case["inter"]
        out = [(case["vocab"], w)]
        for _ in range(case["layers"]):
            out += [(w, w), (kv, w), (kv, w), (w, w), (inter, w), (inter, w), (w, inter), (w,), (w,)]
        out += [(w,), (case["vocab"], w)]
    else:  # ragged: odd matrices and vectors, every 17th tensor empty
        r, side = random.Random(case["mix"]), case["side"]
        for i in range(case["tensors"]):
            a, b = r.randint(max(1, side // 4), side), r.randint(max(1, side // 4), side)
            out.append((0, b) if i % 17 == 16 else (a, b) if i % 3 else (4 * a + 1,))
    return out


def _types(case):
    """One element type per tensor: vectors of a ragged 16-bit set are float32."""
    small = case["net"] == "ragged" and case["dtype"] != "f32"
    return ["f32" if small and len(s) == 1 else case["dtype"] for s in _shapes(case)]


def _out_types(case):
    return _types(case) if case["out"] in (None, "same") else [case["out"]] * len(_shapes(case))


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _buffers(case, types):
    """Tensors of the case's shapes as views of one flat zeroed buffer per element type, as a
    program that buckets its gradients holds them (a ragged set's follow each other without a
    gap, so that most start off any alignment); the buffers too."""
    shapes = _shapes(case)
    gap = 1 if case["net"] == "ragged" else ALIGN
    room = [-(-math.prod(s) // gap) * gap for s in shapes]
    flat = {t: torch.zeros(sum(n for n, u in zip(room, types) if u == t), dtype=DTYPES[t], device="cuda")
            for t in sorted(set(types))}
    at, views = dict.fromkeys(flat, 0), []
    for s, n, t in zip(shapes, room, types):
        views.append(flat[t][at[t]:at[t] + math.prod(s)].view(s))
        at[t] += n
    return views, flat


def _gradients(case, seed):
    """Normal values times a scale per tensor, log-uniform over what backward passes leave."""
    g, r = _gen(seed), random.Random(seed)
    views, flat = _buffers(case, _types(case))
    for x in views:
        x.normal_(generator=g).mul_(2.0 ** r.randint(-13, -7))
    return views, flat


def _head(case, seed):
    """Hidden states that partly point at their target's row, as a trained model's do, an
    output matrix of normal rows, and targets of which the frequent ones come first."""
    g = _gen(seed)
    n, v, d = case["n"], case["v"], case["d"]
    dt = DTYPES[case["dtype"]]
    w = torch.empty(v, d, dtype=dt, device="cuda").normal_(generator=g).mul_(0.02)
    u = torch.rand(n, device="cuda", generator=g)
    y = (torch.exp(u * math.log(v + 1.0)) - 1.0).long().clamp(0, v - 1)
    h = torch.randn(n, d, device="cuda", generator=g)
    rows = w[y].float()
    pull = 12.0 * torch.rand(n, 1, device="cuda", generator=g)
    h += rows * (pull / rows.square().sum(1, keepdim=True).clamp(min=1e-12))
    if case["ignored"]:
        y[torch.randperm(n, device="cuda", generator=g)[:case["ignored"]]] = IGNORE
    return h.to(dt), w, y


def prepare(case, seed):
    state = {"case": case}
    if case["kind"] in ("norm", "clip"):
        state["grads"], state["flat"] = _gradients(case, seed)
        if case["kind"] == "clip" and case["out"] is not None:
            state["out"], state["flat"] = _buffers(case, _out_types(case))
        return state
    h, w, y = _head(case, seed)
    if case["kind"] == "train":
        h.requires_grad_(True)
        w.requires_grad_(True)
        state["grad_loss"] = torch.tensor(case["scale"], device="cuda")
    state.update(hidden=h, weight=w, targets=y)
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    from gefen_amd import clip_gradients, gradient_norm, linear_cross_entropy

    case = state["case"]
    if case["kind"] == "norm":
        return gradient_norm(state["grads"])
    if case["kind"] == "clip":
        total = clip_gradients(state["grads"], case["max_norm"], out=state.get("out"))
        return {"norm": total, "grads": state["flat"]}
    h, w, y = state["hidden"], state["weight"], state["targets"]
    if case["kind"] == "eval":
        with torch.no_grad():
            return linear_cross_entropy(h, w, y, ignore_index=IGNORE, label_smoothing=case["smoothing"],
                                        reduction="none")
    loss = linear_cross_entropy(h, w, y, ignore_index=IGNORE, label_smoothing=case["smoothing"])
    dh, dw = torch.autograd.grad(loss, (h, w), grad_outputs=state["grad_loss"])
    return {"loss": loss.detach(), "dhidden": dh, "dweight": dw}


def _run_plain(state):
    case = state["case"]
    if case["kind"] in ("norm", "clip"):
        total = torch.zeros((), device="cuda")
        for g in state["grads"]:
            total = total + g.float().square().sum()
        total = total.sqrt()
        if case["kind"] == "norm":
            return total
        coef = (case["max_norm"] / (total + EPS)).clamp(max=1.0)
        out = state.get("out", state["grads"])
        for g, o in zip(state["grads"], out):
            o.copy_(g.float() * coef)
        return {"norm": total, "grads": state["flat"]}
    with torch.no_grad():
        h, w, y = state["hidden"].float(), state["weight"].float(), state["targets"]
        v, e = case["v"], case["smoothing"]
        valid = y != IGNORE
        at = y.clamp(min=0)[:, None]
        logits = h @ w.t()
        top = logits.amax(1, keepdim=True)
        p = (logits - top).exp()
        z = p.sum(1, keepdim=True)
        rows = (top + z.log() - (1.0 - e) * logits.gather(1, at))[:, 0]
        if e:
            rows = rows - (e / v) * logits.sum(1)
        rows = torch.where(valid, rows, torch.zeros_like(rows))
        if case["kind"] == "eval":
            return rows
        del logits
        count = valid.sum()
        p = p / z
        p.scatter_add_(1, at, torch.full_like(z, e - 1.0))
        if e:
            p = p - e / v
        p = p * (valid[:, None] * (state["grad_loss"] / count))
        dt = DTYPES[case["dtype"]]
        return {"loss": rows.sum() / count, "dhidden": (p @ w).to(dt), "dweight": (p.t() @ h).to(dt)}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] in ("norm", "clip"):
        sizes = [math.prod(s) for s in _shapes(case)]
        nbytes = sum(n * SIZE[t] for n, t in zip(sizes, _types(case))) + 4
        flops = 2 * sum(sizes)
        if case["kind"] == "clip" and case["out"] is not None:
            nbytes += sum(n * SIZE[t] for n, t in zip(sizes, _out_types(case)))
            flops += sum(sizes)
        return {"bytes": nbytes, "flops": flops}
    n, v, d, size = case["n"], case["v"], case["d"], SIZE[case["dtype"]]
    rows = n - case["ignored"]
    if case["kind"] == "eval":
        return {"bytes": (rows + v) * d * size + 12 * n, "flops": 2 * rows * v * d}
    return {"bytes": (rows + v) * d * size + 8 * n + (n + v) * d * size + 4, "flops": 6 * rows * v * d}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    if case["kind"] in ("norm", "clip"):
        grads, _ = _gradients(case, seed)
        total = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g.double())) ** 2 for g in grads if g.numel()))
        norm = torch.tensor(total, dtype=torch.float64, device="cuda")
        if case["kind"] == "norm":
            return norm
        coef = min(1.0, case["max_norm"] / (total + EPS))
        types = _out_types(case)
        gap = 1 if case["net"] == "ragged" else ALIGN
        flat = {}
        for t in sorted(set(types)):
            parts = []
            for g in (g for g, u in zip(grads, types) if u == t):
                parts += [g.double().reshape(-1) * coef, g.new_zeros(-g.numel() % gap, dtype=torch.float64)]
            flat[t] = torch.cat(parts)
        return {"norm": norm, "grads": flat}
    h, w, y = (t.detach() for t in _head(case, seed))
    n, v, e = case["n"], case["v"], case["smoothing"]
    w = w.double()
    rows = torch.zeros(n, dtype=torch.float64, device="cuda")
    train = case["kind"] == "train"
    if train:
        factor = case["scale"] / int((y != IGNORE).sum())
        dh = torch.zeros(h.shape, dtype=torch.float64, device="cuda")
        dw = torch.zeros(w.shape, dtype=torch.float64, device="cuda")
    live = torch.nonzero(y != IGNORE)[:, 0]
    for part in live.split(2048):
        x, t = h[part].double(), y[part]
        logits = torch.mm(x, w.t())
        logp = logits - torch.logsumexp(logits, dim=1)[:, None]
        rows[part] = -(1.0 - e) * logp[torch.arange(len(part), device="cuda"), t] - e * logp.mean(1)
        if train:
            q = torch.full_like(logp, e / v)
            q[torch.arange(len(part), device="cuda"), t] += 1.0 - e
            diff = (logp.exp() - q) * factor
            dh[part] = torch.mm(diff, w)
            dw += torch.mm(diff.t(), x)
    if not train:
        return rows
    return {"loss": rows.sum() / len(live), "dhidden": dh, "dweight": dw}
