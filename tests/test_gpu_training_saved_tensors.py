"""What waits for backward is seen by the hooks of saved tensors: it can be offloaded, and
checkpointing frees it."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,limit", [(torch.float16, None), (torch.bfloat16, None), (torch.bfloat16, 1 << 20),
                                         (torch.float32, None)])
def test_what_waits_for_backward_can_be_offloaded(dtype, limit):
    from gefen_amd import linear_cross_entropy

    g = torch.Generator().manual_seed(2)
    h = torch.randn(1000, 64, generator=g).cuda().to(dtype).requires_grad_(True)
    w = (torch.randn(4096, 64, generator=g) * 0.2).cuda().to(dtype).requires_grad_(True)
    y = torch.randint(0, 4096, (1000,), generator=g).cuda()
    want = torch.autograd.grad(linear_cross_entropy(h, w, y, workspace_limit=limit), (h, w))
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with torch.autograd.graph.save_on_cpu():
        loss = linear_cross_entropy(h, w, y, workspace_limit=limit)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() - before <= 4096
    got = torch.autograd.grad(loss, (h, w), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    again = torch.autograd.grad(loss, (h, w))  # of a retained graph: from the operands
    for a, b in zip(again, want):
        assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -7, atol=1e-6)


def test_checkpointing_frees_what_waits_for_backward():
    from torch.utils.checkpoint import checkpoint

    from gefen_amd import linear_cross_entropy

    torch.manual_seed(3)
    h = torch.randn(1000, 64, device="cuda").half().requires_grad_(True)
    w = (torch.randn(4096, 64, device="cuda") * 0.2).half().requires_grad_(True)
    y = torch.randint(0, 4096, (1000,), device="cuda")
    want = torch.autograd.grad(linear_cross_entropy(h, w, y), (h, w))
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    loss = checkpoint(linear_cross_entropy, h, w, y, use_reentrant=False)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() - before <= 4096
    got = torch.autograd.grad(loss, (h, w))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
