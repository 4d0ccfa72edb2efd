"""Many short problems: more (batch, key head) pairs than one pass of 16 workgroups each could launch."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
F = 2.0 ** -24


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_a_million_windows(dtype):
    """2^20 + 2 heads of one query over one key: the output is the value and the value's gradient the
    output's, times a probability of 1 that is off by delta (test_gpu_attention, n = 1) in the product
    and in L; in 16 bits that is far below a rounding and rounds to the value itself.  dS = dO v - D
    is zero but for two sums of d products, D's output being off by the same, and in float16 for half
    the spacing 2^-39 of its bound 4 |dO| max |v|."""
    from gefen_amd import attention

    g = torch.Generator(device="cuda").manual_seed(5)
    b, hk, d = (1 << 19) + 1, 2, 8
    q, k, v, go = (torch.randn(b, 1, hk, d, device="cuda", generator=g).to(DT[dtype]) for _ in range(4))
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = attention(*leaves)
    dq, dk, dv = torch.autograd.grad(out, leaves, grad_outputs=go)
    if dtype != "f32":
        assert torch.equal(out.detach(), v) and torch.equal(dv, go)
    q, k, v, go = (t.double() for t in (q, k, v, go))
    scores = d ** -0.5 * (q * k).abs().sum(-1, keepdim=True)
    off = 2 * (d + 4) * F * scores + 34 * F + 8 * F * scores + 6 * F  # delta, (n + 4) f and the result's own
    if dtype == "f32":
        assert bool(((out.double() - v).abs() <= off * v.abs()).all())
        assert bool(((dv.double() - go).abs() <= off * go.abs()).all())
    ds = (2 * (d + 4) * F + off) * (go * v).abs().sum(-1, keepdim=True)
    if dtype == "f16":
        ds = ds + 2.0 ** -39 * 4 * go.norm(dim=-1, keepdim=True) * v.norm(dim=-1, keepdim=True)
    # dS is rounded to 16 bits and so are the gradients (float16: half the subnormal spacing): twice its size covers both
    tiny = 2.0 ** -25 if dtype == "f16" else 0.0
    for got, other in ((dq, k), (dk, q)):
        assert bool((got.double().abs() <= 2 * d ** -0.5 * ds * other.abs() + tiny).all())
