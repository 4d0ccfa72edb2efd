"""The operators of a layer in a training step beside its matrix products, as timed cases.

Three operators, through the public entry points:

* ``attention``: softmax attention with shared key heads, causal or not, over padded batches
  or packed sequences, with its gradients (``train``) or without (``eval``);
* ``norm``: the root-mean-square norm of a residual stream with the addition before it,
  with gradients (``train``), or with an output in 8 bits and scales (``eight``);
* ``dropout``: from a counter-based generator, alone or added to a residual, with its
  gradient.

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
E4M3_MAX = 448.0
EPS = 1e-6


# ------------------------------------------------------------------ cases
def listed():
    return [
        # a test-sized float32 model's attention: all latency
        {"name": "attention small f32", "kind": "attention", "mode": "train", "dtype": "f32", "batch": 2, "queries": 19,
         "keys": 19, "heads": 4, "kv_heads": 4, "width": 24, "causal": True, "padded": False, "packed": 0},
        # answering: one new token of each of 16 sequences of uneven length
        {"name": "attention one token bf16", "kind": "attention", "mode": "eval", "dtype": "bf16", "batch": 16,
         "queries": 1, "keys": 8192, "heads": 32, "kv_heads": 8, "width": 128, "causal": False, "padded": True,
         "packed": 0},
        # eight sequences of 1024 through a float32 GPT-2 layer
        {"name": "attention gpt2 f32", "kind": "attention", "mode": "train", "dtype": "f32", "batch": 8,
         "queries": 1024, "keys": 1024, "heads": 12, "kv_heads": 12, "width": 64, "causal": True, "padded": False,
         "packed": 0},
        # float16, a padded batch that looks at another one (an encoder's output), sizes that divide badly
        {"name": "attention odd f16", "kind": "attention", "mode": "train", "dtype": "f16", "batch": 5, "queries": 777,
         "keys": 1003, "heads": 6, "kv_heads": 3, "width": 80, "causal": False, "padded": True, "packed": 0},
        # a micro-batch of 16384 tokens in documents of uneven length, 1.5B shapes
        {"name": "attention packed llama1.5b bf16", "kind": "attention", "mode": "train", "dtype": "bf16", "batch": 1,
         "queries": 16384, "keys": 16384, "heads": 32, "kv_heads": 8, "width": 64, "causal": True, "padded": False,
         "packed": 11},
        # one long sequence through an 8B layer: the largest
        {"name": "attention llama8b bf16", "kind": "attention", "mode": "train", "dtype": "bf16", "batch": 1,
         "queries": 8192, "keys": 8192, "heads": 32, "kv_heads": 8, "width": 128, "causal": True, "padded": False,
         "packed": 0},
        # a test-sized model's norm: all latency
        {"name": "norm small f32", "kind": "norm", "mode": "train", "dtype": "f32", "rows": 48, "width": 96,
         "residual": True, "dropout": 0.0},
        # the residual stream of 8192 tokens of an 8B model
        {"name": "norm llama8b bf16", "kind": "norm", "mode": "train", "dtype": "bf16", "rows": 8192, "width": 4096,
         "residual": True, "dropout": 0.0},
        # float16 rows of odd width, with the residual's dropout
        {"name": "norm odd f16", "kind": "norm", "mode": "train", "dtype": "f16", "rows": 1531, "width": 1001,
         "residual": True, "dropout": 0.1},
        # evaluation with 8-bit inputs of the next product, 1.5B shapes
        {"name": "norm 8 bit llama1.5b bf16", "kind": "norm", "mode": "eight", "dtype": "bf16", "rows": 16384,
         "width": 2048, "residual": True, "dropout": 0.0},
        # the residual dropout of a float32 GPT-2 layer
        {"name": "dropout gpt2 f32", "kind": "dropout", "dtype": "f32", "rows": 8192, "width": 768, "residual": True,
         "p": 0.1},
        # the inner activations of 16384 tokens of an 8B model: the largest
        {"name": "dropout llama8b bf16", "kind": "dropout", "dtype": "bf16", "rows": 16384, "width": 14336,
         "residual": False, "p": 0.1},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed ones' ranges, at most as large as the largest of its kind."""
    kind = rng.choice(["attention", "attention", "attention", "norm", "norm", "dropout"])
    case = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if kind == "norm":
        while True:
            rows, width = _spread(rng, 1, 65536), _spread(rng, 3, 16384)
            if rows * width <= 8192 * 4096:
                break
        mode = rng.choice(["train", "train", "eight"])
        residual = rng.random() < 0.7
        case.update(mode=mode, rows=rows, width=-(-width // 8) * 8 if rng.random() < 0.5 else width, residual=residual,
                    dropout=rng.choice([0.0, 0.0, 0.1, 0.5]) if residual and mode == "train" else 0.0)
        return case
    if kind == "dropout":
        while True:
            rows, width = _spread(rng, 1, 65536), _spread(rng, 3, 16384)
            if rows * width <= 16384 * 14336:
                break
        case.update(rows=rows, width=width, residual=rng.random() < 0.5, p=rng.choice([0.05, 0.1, 0.1, 0.3, 0.5]))
        return case
    mode = rng.choice(["train", "train", "eval"])
    layout = rng.choice(["plain", "plain", "cross", "packed", "token"])
    causal = layout != "cross" and rng.random() < 0.7
    while True:
        kv, group = rng.choice([1, 2, 3, 4, 8, 12]), rng.choice([1, 1, 2, 3, 4, 8])
        width = rng.choice([16, 24, 40, 64, 64, 80, 96, 128, 128, rng.randint(8, 128)])
        batch, queries = _spread(rng, 1, 32), _spread(rng, 1, 8192)
        keys = queries
        if layout == "cross":
            keys = _spread(rng, 1, 8192)
        elif layout == "packed":
            batch = 1
        elif layout == "token":
            mode, keys, queries = "eval", queries, rng.choice([1, 1, 2, 5])
        pairs = batch * queries * keys * kv * group
        limit = 8192 * 8192 * 32 * 128 // 2 // (1 if case["dtype"] != "f32" else 16)
        if pairs * width <= limit and pairs <= 1 << 30:
            break
    case.update(mode=mode, batch=batch, queries=queries, keys=keys, heads=kv * group, kv_heads=kv, width=width,
                causal=causal, padded=layout in ("cross", "token") or (layout == "plain" and rng.random() < 0.3),
                packed=rng.randint(1, 12) if layout == "packed" else 0)
    return case


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _documents(case):
    """Lengths of the packed sequences: uneven, the first of a single token where there are
    several; they fill the tokens."""
    r, n = random.Random(case["packed"]), case["packed"]
    cuts = sorted(r.randint(1, case["queries"]) for _ in range(n - 1))
    if cuts:
        cuts[0] = 1
    at = [0] + cuts + [case["queries"]]
    return [b - a for a, b in zip(at, at[1:])]


def _key_lengths(case, seed):
    """Keys of each sequence of a padded batch: uneven; one of several sequences has none."""
    r, s = random.Random(seed), case["keys"]
    lengths = [r.randint(max(1, s // 2), s) for _ in range(case["batch"])]
    if case["batch"] >= 4:
        lengths[r.randrange(case["batch"])] = 0
    return lengths


def _attention_inputs(case, seed):
    """Queries, keys and values as a model's projections leave them: views of one buffer where
    they come of the same tokens; logits of a standard deviation of about 1.5; dO of unit size
    for float16 (scaled losses), else small."""
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    b, sq, sk, h, hk, d = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "width"))
    if sq == sk and not case["padded"]:
        buf = torch.randn(b, sq, (h + 2 * hk) * d, device="cuda", generator=g)
        buf[..., :h * d] *= 1.5
        buf = buf.to(dt)
        q, k, v = (x.unflatten(-1, (-1, d)) for x in buf.split([h * d, hk * d, hk * d], dim=-1))
    else:
        q = (1.5 * torch.randn(b, sq, h, d, device="cuda", generator=g)).to(dt)
        k = torch.randn(b, sk, hk, d, device="cuda", generator=g).to(dt)
        v = torch.randn(b, sk, hk, d, device="cuda", generator=g).to(dt)
    do = torch.randn(b, sq, h, d, device="cuda", generator=g)
    do = (do if case["dtype"] == "f16" else do * 2.0 ** -10).to(dt)
    if case["packed"]:
        q, k, v, do = q[0], k[0], v[0], do[0]
    return q, k, v, do


def _rows_inputs(case, seed):
    """A branch's output, the residual stream it joins (larger, with a few strong channels) and
    gradients of both outputs."""
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    shape = (case["rows"], case["width"])
    x = torch.randn(shape, device="cuda", generator=g).to(dt)
    res = torch.randn(shape, device="cuda", generator=g) * 3.0
    res[:, ::97] *= 8.0
    res = res.to(dt) if case["residual"] else None
    w = (1.0 + 0.2 * torch.randn(case["width"], device="cuda", generator=g)).to(dt)
    down = 1.0 if case["dtype"] == "f16" else 2.0 ** -10
    dy = (down * torch.randn(shape, device="cuda", generator=g)).to(dt)
    ds = (down * torch.randn(shape, device="cuda", generator=g)).to(dt)
    return x, res, w, dy, ds


def _seed_of(seed):
    return (seed * 0x9E3779B97F4A7C15 + 1) % (1 << 63)


def prepare(case, seed):
    state = {"case": case}
    if case["kind"] == "attention":
        q, k, v, do = _attention_inputs(case, seed)
        if case["padded"]:
            state["key_lengths"] = torch.tensor(_key_lengths(case, seed), dtype=torch.int32, device="cuda")
        if case["packed"]:
            lengths = _documents(case)
            state["documents"] = lengths
            state["offsets"] = torch.tensor([0] + lengths, device="cuda").cumsum(0).to(torch.int32)
        if case["mode"] == "train":
            for t in (q, k, v):
                t.requires_grad_(True)
            state["grad"] = do
        state.update(query=q, key=k, value=v)
        return state
    x, res, w, dy, ds = _rows_inputs(case, seed)
    if case["kind"] == "dropout" or case["mode"] == "train":
        for t in (x, res) if case["kind"] == "dropout" else (x, res, w):
            if t is not None:
                t.requires_grad_(True)
    if case.get("p") or case.get("dropout"):
        state["seed"] = torch.tensor(_seed_of(seed), dtype=torch.int64, device="cuda")  # a program counts it up
        state["offset"] = 3 + seed % 5                                                  # the layer's place
    state.update(x=x, residual=res, weight=w, grad=dy, grad_sum=ds)
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    import gefen_amd

    case = state["case"]
    if case["kind"] == "attention":
        q, k, v = state["query"], state["key"], state["value"]
        if case["mode"] == "eval":
            with torch.no_grad():
                return gefen_amd.attention(q, k, v, causal=case["causal"], key_lengths=state.get("key_lengths"),
                                           offsets=state.get("offsets"))
        out = gefen_amd.attention(q, k, v, causal=case["causal"], key_lengths=state.get("key_lengths"),
                                  offsets=state.get("offsets"))
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), grad_outputs=state["grad"])
        return {"out": out.detach(), "dquery": dq, "dkey": dk, "dvalue": dv}
    x, res = state["x"], state["residual"]
    if case["kind"] == "dropout":
        y = gefen_amd.dropout(x, case["p"], state["seed"], offset=state["offset"], residual=res)
        dx, = torch.autograd.grad(y, (x,), grad_outputs=state["grad"])
        return {"y": y.detach(), "dx": dx}
    w = state["weight"]
    if case["mode"] == "eight":
        with torch.no_grad():
            q, scales, *s = gefen_amd.rms_norm_quantized(x, w, eps=EPS, residual=res)
            return {"y": q, "scales": scales, "sum": s}
    y = gefen_amd.rms_norm(x, w, eps=EPS, residual=res, dropout=case["dropout"], seed=state.get("seed"),
                           offset=state.get("offset", 0))
    if res is None:
        dx, dw = torch.autograd.grad(y, (x, w), grad_outputs=state["grad"])
        return {"y": y.detach(), "dx": dx, "dweight": dw}
    y, s = y
    dx, dr, dw = torch.autograd.grad((y, s), (x, res, w), grad_outputs=(state["grad"], state["grad_sum"]))
    return {"y": y.detach(), "sum": s.detach(), "dx": dx, "dresidual": dr, "dweight": dw}


def _plain_attention(q, k, v, causal, key_lengths, do):
    """[B, S, H, D] operands of one dtype; the output, and the gradients where do is given."""
    dt, (b, sq, h, d), (sk, hk) = q.dtype, q.shape, k.shape[1:3]
    scale, group = d ** -0.5, h // hk

    def rows(t):  # [B * Hk, group * Sq, D]
        return t.float().transpose(1, 2).reshape(b * hk, -1, d)

    q32, k32, v32 = rows(q), rows(k), rows(v)
    j = torch.arange(sk, device=q.device)
    seen = torch.ones(1, 1, 1, sk, dtype=torch.bool, device=q.device)
    if causal:
        i = torch.arange(sq, device=q.device)[:, None]
        seen = seen & (j <= i + (sk - sq))[None, None]
    if key_lengths is not None:
        seen = seen & (j < key_lengths[:, None])[:, None, None]
    s = (torch.bmm(q32, k32.transpose(1, 2).contiguous()) * scale).view(b, h, sq, sk)
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = (s - torch.where(top == -math.inf, torch.zeros_like(top), top)).exp()
    del s
    z = p.sum(-1, keepdim=True)
    p = (p / torch.where(z == 0, torch.ones_like(z), z)).view(b * hk, group * sq, sk)
    o = torch.bmm(p, v32)

    def back(t, heads):
        return t.view(b, heads, -1, d).transpose(1, 2).to(dt)

    if do is None:
        return back(o, h)
    do32 = rows(do)
    dv = torch.bmm(p.transpose(1, 2).contiguous(), do32)
    ds = torch.bmm(do32, v32.transpose(1, 2).contiguous())
    ds = p * (ds - (do32 * o).sum(-1, keepdim=True))
    del p
    dq = torch.bmm(ds, k32) * scale
    dk = torch.bmm(ds.transpose(1, 2).contiguous(), q32) * scale
    return back(o, h), back(dq, h), back(dk, hk), back(dv, hk)


def _plain_keep(shape, p, seed, offset, device):
    """The dropout's factors: Philox4x32-10 (Salmon et al., 2011) on (element / 8, offset)."""
    n = math.prod(shape)
    low = 0xFFFFFFFF
    block = torch.arange(-(-n // 8), device=device)
    c = [block & low, block >> 32, torch.full_like(block, offset & low), torch.full_like(block, offset >> 32)]
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & low) ^ c[1] ^ k0, b & low, ((a >> 32) & low) ^ c[3] ^ k1, a & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack(c, 1)
    u = torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:n]
    cut = round(p * 65536)
    return (u >= cut).float().view(shape) * (65536.0 / (65536 - cut))


def _run_plain(state):
    case = state["case"]
    with torch.no_grad():
        if case["kind"] == "attention":
            q, k, v, do = state["query"], state["key"], state["value"], state.get("grad")
            if case["packed"]:
                parts, at = [], 0
                for n in state["documents"]:
                    if n:
                        part = [None if t is None else t[at:at + n][None] for t in (q, k, v, do)]
                        parts.append(_plain_attention(*part[:3], case["causal"], None, part[3]))
                    at += n
                if do is None:
                    return torch.cat(parts, 1)[0]
                res = [torch.cat(t, 1)[0] for t in zip(*parts)]
            else:
                lengths = state.get("key_lengths")
                # as many sequences at a time as 2^30 probabilities hold
                step = max(1, (1 << 30) // (case["heads"] * case["queries"] * case["keys"]))
                parts = [_plain_attention(*(t[b:b + step] for t in (q, k, v)), case["causal"],
                                          None if lengths is None else lengths[b:b + step],
                                          None if do is None else do[b:b + step])
                         for b in range(0, case["batch"], step)]
                if do is None:
                    return torch.cat(parts)
                res = [torch.cat(t) for t in zip(*parts)]
            return dict(zip(("out", "dquery", "dkey", "dvalue"), res))
        x, res = state["x"], state["residual"]
        dt, p = x.dtype, case.get("p") or case.get("dropout") or 0.0
        keep = _plain_keep(x.shape, p, state["seed"], state["offset"], x.device) if p else 1.0
        s = x.float() * keep
        if res is not None:
            s = s + res.float()
        if case["kind"] == "dropout":
            return {"y": s.to(dt), "dx": (state["grad"].float() * keep).to(dt)}
        w = state["weight"].float()
        r = torch.rsqrt(s.square().mean(-1, keepdim=True) + EPS)
        y = s * r * w
        if case["mode"] == "eight":
            c = y.abs().amax(-1, keepdim=True) / E4M3_MAX
            q = (y / torch.where(c > 0, c, torch.ones_like(c))).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
            return {"y": q, "scales": c[:, 0], "sum": [] if res is None else [s.to(dt)]}
        dy = state["grad"].float()
        n = s * r
        g = dy * w
        out = {"y": y.to(dt)}
        dsum = r * (g - n * (g * n).mean(-1, keepdim=True))
        if res is not None:
            out["sum"] = s.to(dt)
            dsum = dsum + state["grad_sum"].float()
        out["dx"] = (dsum * keep).to(dt)
        if res is not None:
            out["dresidual"] = dsum.to(dt)
        out["dweight"] = (dy * n).sum(0).to(dt)
        return out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = SIZE[case["dtype"]]
    if case["kind"] == "attention":
        b, sq, sk, h, hk, d = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "width"))

        def pairs(n, m):  # of n queries and m keys, the last query at the last key
            if not case["causal"]:
                return n * m
            return sum(max(0, i + 1) for i in range(m - n, m)) if n <= m else m * (m + 1) // 2

        if case["packed"]:
            p = sum(pairs(n, n) for n in _documents(case))
            rows, keys = sq, sk
        elif case["padded"]:
            lengths = _key_lengths(case, 0)  # any seed's: the lengths are of one distribution
            p = sum(min(pairs(sq, sk), sq * n) for n in lengths)
            rows, keys = b * sq, sum(lengths)
        else:
            p, rows, keys = b * pairs(sq, sk), b * sq, b * sk
        q_bytes, kv_bytes = rows * h * d * size, keys * hk * d * size
        if case["mode"] == "eval":
            return {"bytes": 2 * q_bytes + 2 * kv_bytes, "flops": 4 * p * h * d}
        return {"bytes": 4 * q_bytes + 4 * kv_bytes, "flops": 14 * p * h * d}
    n = case["rows"] * case["width"]
    res = 1 if case["residual"] else 0
    if case["kind"] == "dropout":
        return {"bytes": (2 + res + 2) * n * size, "flops": 2 * (1 + res + 1) * n}
    if case["mode"] == "eight":
        return {"bytes": (1 + 2 * res) * n * size + n + case["width"] * size + 4 * case["rows"], "flops": 8 * n}
    outs = 2 if case["dropout"] else 1  # of the two gradients, equal without dropout
    tensors = (1 + res) + (1 + res) + (1 + res) + outs  # in, out, gradients in, gradients out
    return {"bytes": tensors * n * size + 2 * case["width"] * size, "flops": 16 * n}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_sequence(q, k, v, seen, do):
    """One sequence and key head: q [G, n, D], k and v [m, D], seen [n, m]."""
    q, k, v = (t.double().requires_grad_(do is not None) for t in (q, k, v))
    with torch.enable_grad():
        outs = []
        for one in q.unbind(0):
            logits = torch.mm(one, k.t()) / math.sqrt(one.shape[-1])
            logits = torch.where(seen, logits, logits.new_tensor(-math.inf))
            total = torch.logsumexp(logits, 1, keepdim=True)
            total = torch.where(seen.any(1, keepdim=True), total, total.new_zeros(()))
            outs.append(torch.mm(torch.exp(logits - total), v))
        out = torch.stack(outs)
    if do is None:
        return (out,)
    return (out.detach(),) + torch.autograd.grad(out, (q, k, v), grad_outputs=do.double())


def _exact_attention(case, seed):
    q, k, v, do = (t.detach() for t in _attention_inputs(case, seed))
    train, group = case["mode"] == "train", case["heads"] // case["kv_heads"]
    res = [torch.zeros(t.shape, dtype=torch.float64, device=t.device) for t in (q, q, k, v)]
    if case["packed"]:
        ends = torch.tensor(_documents(case)).cumsum(0).tolist()
        places = [(slice(a, e), slice(a, e), ()) for a, e in zip([0] + ends, ends)]
    else:
        lengths = _key_lengths(case, seed) if case["padded"] else [case["keys"]] * case["batch"]
        places = [(slice(None), slice(0, n), (b,)) for b, n in enumerate(lengths)]
    for rows, keys, at in places:
        a, b = q[at][rows], k[at][keys]
        if not a.shape[0] or not b.shape[0]:
            continue
        seen = torch.ones(a.shape[0], b.shape[0], dtype=torch.bool, device=q.device)
        if case["causal"]:
            seen = seen.tril(0 if case["packed"] else case["keys"] - case["queries"])
        for head in range(case["kv_heads"]):
            own_heads = slice(head * group, (head + 1) * group)
            got = _exact_sequence(a[:, own_heads].transpose(0, 1), b[:, head], v[at][keys][:, head], seen,
                                  do[at][rows][:, own_heads].transpose(0, 1) if train else None)
            res[0][at][rows, own_heads] = got[0].transpose(0, 1)
            if train:
                res[1][at][rows, own_heads] = got[1].transpose(0, 1)
                res[2][at][keys, head] = got[2]
                res[3][at][keys, head] = got[3]
    return dict(zip(("out", "dquery", "dkey", "dvalue"), res)) if train else res[0]


def _exact_keep(shape, p, seed, offset):
    """The same factors with the products in 16-bit halves of the multipliers."""
    n, mask = math.prod(shape), (1 << 32) - 1
    i = torch.arange((n + 7) // 8, dtype=torch.int64, device="cuda")

    def times(x, m):
        lo, hi = x * (m & 0xFFFF), x * (m >> 16)       # below 2^48
        mid = hi + (lo >> 16)
        return mid >> 16, ((mid & 0xFFFF) << 16) | (lo & 0xFFFF)

    x0, x1 = i & mask, i >> 32
    x2, x3 = torch.zeros_like(i) + (offset & mask), torch.zeros_like(i) + (offset >> 32)
    for r in range(10):
        key0, key1 = ((seed & mask) + r * 0x9E3779B9) & mask, ((seed >> 32) + r * 0xBB67AE85) & mask
        h0, l0 = times(x0, 0xD2511F53)
        h2, l2 = times(x2, 0xCD9E8D57)
        x0, x1, x2, x3 = h2 ^ x1 ^ key0, l2, h0 ^ x3 ^ key1, l0
    u = torch.empty(i.numel(), 8, dtype=torch.int64, device="cuda")
    for w, x in enumerate((x0, x1, x2, x3)):
        u[:, 2 * w] = x & 0xFFFF
        u[:, 2 * w + 1] = x >> 16
    cut = int(round(p * 65536))
    kept = u.view(-1)[:n].view(shape) >= cut
    return kept.double() / (1.0 - cut / 65536.0)


def exact(case, seed):
    if case["kind"] == "attention":
        return _exact_attention(case, seed)
    x, res, w, dy, ds = _rows_inputs(case, seed)
    p = case.get("p") or case.get("dropout") or 0.0
    s = x.double()
    keep = _exact_keep(x.shape, p, _seed_of(seed), 3 + seed % 5) if p else None
    if keep is not None:
        s = s * keep
    if res is not None:
        s = s + res.double()
    if case["kind"] == "dropout":
        return {"y": s, "dx": dy.double() * keep}
    w = w.double()
    size = torch.sqrt((s * s).sum(1, keepdim=True) / case["width"] + EPS)
    n = s / size
    y = n * w
    if case["mode"] == "eight":
        c = y.abs().amax(1) / E4M3_MAX
        return {"y": y / c.clamp(min=1e-300)[:, None], "scales": c, "sum": [] if res is None else [s]}
    g = dy.double() * w
    dsum = (g - n * ((g * n).sum(1, keepdim=True) / case["width"])) / size
    out = {"y": y, "dweight": (dy.double() * n).sum(0)}
    if res is not None:
        dsum = dsum + ds.double()
        out["sum"], out["dresidual"] = s, dsum
    out["dx"] = dsum if keep is None else dsum * keep
    return out
