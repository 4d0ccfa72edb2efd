"""Attention: large finite values in rows that take no part, and operands of a task that run backwards."""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BIG = 6.0e4  # finite in float16, and so is the norm of a row of it


def call(q, k, v, go, **kw):
    from gefen_amd import attention

    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = attention(q, k, v, **kw)
    return (out.detach(),) + torch.autograd.grad(out, (q, k, v), grad_outputs=go)


def make(dtype, b, sq, sk, h, hk, d, seed=0):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(b, s, n, d, generator=g).to(DT[dtype]).cuda() * f
                 for s, n, f in ((sq, h, 1.0), (sk, hk, 1.0), (sk, hk, 2.0 ** -8), (sq, h, 2.0 ** -8)))


def same(a, b):
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", list(DT))
def test_rows_outside_of_the_packed_sequences(dtype):
    """Rows in front of the first sequence and behind the last one: gradients are those of zeros there, bit for bit."""
    q, k, v, go = (t[0] for t in make(dtype, 1, 300, 300, 4, 2, 64))
    offsets = torch.tensor([40, 41, 170, 230], dtype=torch.int32, device="cuda")
    results = []
    for value in (0.0, BIG):
        w, g = v.clone(), go.clone()
        for t in (w, g):
            t[:40] = value
            t[230:] = value
        results.append(call(q, k, w, g, causal=True, offsets=offsets))
    same(*results)
    assert float(results[0][1].abs().max()) > 0


@pytest.mark.parametrize("dtype", list(DT))
def test_queries_that_see_nothing(dtype):
    """A causal query in front of the first key, and a sequence without keys."""
    q, k, v, go = make(dtype, 3, 200, 90, 4, 2, 64)
    lengths = torch.tensor([90, 0, 33], device="cuda")
    results = []
    for value in (0.0, BIG):
        w, g = v.clone(), go.clone()
        g[:, :110] = value
        g[1] = value
        w[1] = value
        w[2, 33:] = value
        results.append(call(q, k, w, g, causal=True, key_lengths=lengths))
    same(*results)
    assert float(results[0][1].abs().max()) > 0


@pytest.mark.parametrize("dtype", list(DT))
def test_a_task_whose_rows_run_backwards(dtype):
    """Negative strides of a task: the results are those of the operands turned round."""
    from gefen_amd import _lib

    b, sq, sk, h, hk, d = 2, 70, 150, 4, 2, 64
    q, k, v, go = make(dtype, b, sq, sk, h, hk, d)
    want = call(q.flip(1).contiguous(), k.flip(1).contiguous(), v.flip(1).contiguous(), go.flip(1).contiguous(), causal=True)
    got = [torch.empty_like(t) for t in want]
    lse = torch.empty(b * sq * h, device="cuda")
    t = _lib.AttentionTask()
    t.out, t.grad_query, t.grad_key, t.grad_value = (x.data_ptr() for x in got)
    t.lse = lse.data_ptr()
    for name, x in (("query", q), ("key", k), ("value", v), ("grad_out", go)):
        setattr(t, name, x[0, -1].data_ptr())
        getattr(t, name + "_strides")[:] = [x.stride(0), -x.stride(1), x.stride(2)]
    t.batch, t.queries, t.keys, t.heads, t.kv_heads, t.width = b, sq, sk, h, hk, d
    t.scale, t.causal, t.dtype = d ** -0.5, 1, {"f32": 0, "f16": 1, "bf16": 2}[dtype]
    lib = _lib.load()
    n = max(int(lib.gefen_attention_forward_workspace_size(ctypes.byref(t))),
            int(lib.gefen_attention_backward_workspace_size(ctypes.byref(t))))
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.gefen_attention_forward(ctypes.byref(t), ws.data_ptr(), n, stream) == 0
    assert lib.gefen_attention_backward(ctypes.byref(t), ws.data_ptr(), n, stream) == 0
    torch.cuda.synchronize()
    # the same sums in the same order, but for how rows are loaded
    same(got, want)
