"""What attention, rms_norm and dropout meet between their forward and backward passes: saved
tensors that come back from hooks in another layout or type, and graph capture beside a graph of
autograd that was recorded outside."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def calls():
    """name -> (leaves, call): each operator with everything that it saves."""
    from gefen_amd import attention, dropout, rms_norm

    g = torch.Generator(device="cuda").manual_seed(5)

    def leaf(*shape):
        return torch.randn(*shape, generator=g, device="cuda").bfloat16().requires_grad_(True)

    q, k, v = leaf(2, 70, 4, 32), leaf(2, 90, 2, 32), leaf(2, 90, 2, 32)
    lengths = torch.tensor([90, 41], device="cuda")
    pq, pk, pv = leaf(70, 4, 32), leaf(70, 2, 32), leaf(70, 2, 32)
    offsets = torch.tensor([0, 33, 64], dtype=torch.int32, device="cuda")
    x, res, w = leaf(50, 6, 72), leaf(50, 6, 72), leaf(72)
    seed = torch.tensor([9], device="cuda")
    return {
        "attention": ((q, k, v), lambda: attention(q, k, v, causal=True, key_lengths=lengths)),
        "packed": ((pq, pk, pv), lambda: attention(pq, pk, pv, offsets=offsets)),
        "norm": ((x, w), lambda: rms_norm(x, w)),
        "sum and norm": ((x, res, w), lambda: rms_norm(x, w, residual=res, dropout=0.3, seed=seed)),
        "dropout": ((x, res), lambda: dropout(x, 0.3, seed, residual=res)),
    }


NAMES = ["attention", "packed", "norm", "sum and norm", "dropout"]


def gradients(name, pack=None):
    leaves, call = calls()[name]
    if pack is None:
        out = call()
    else:
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, pack):
            out = call()
    out = out if isinstance(out, tuple) else (out,)
    g = torch.Generator(device="cuda").manual_seed(6)
    seeds = [torch.randn(o.shape, generator=g, device="cuda").to(o.dtype) for o in out]
    return torch.autograd.grad(out, leaves, grad_outputs=seeds)


def other_layout(t):
    """The same values, every other element of twice the memory, dimensions reversed."""
    wide = torch.zeros(tuple(reversed(t.shape)) + (2,), dtype=t.dtype, device=t.device)
    wide[..., 0] = t.permute(tuple(reversed(range(t.dim()))))
    return wide[..., 0].permute(tuple(reversed(range(t.dim()))))


@pytest.mark.parametrize("name", NAMES)
def test_saved_tensors_may_come_back_in_another_layout(name):
    for a, b in zip(gradients(name), gradients(name, other_layout)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("name", NAMES)
def test_saved_tensors_have_to_keep_their_dtype_and_shape(name):
    for pack in (lambda t: t.double(), lambda t: t.reshape(-1).repeat(2)):
        with pytest.raises(RuntimeError, match="saved tensor"):
            gradients(name, pack)


@pytest.mark.parametrize("name", NAMES)
def test_capture_beside_an_eager_graph_of_the_same_leaves_is_refused(name):
    leaves, call = calls()[name]
    living = call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.zeros(4, device="cuda")
        with pytest.raises(RuntimeError, match="outside the capture"):
            call()
        with torch.no_grad():  # no graph of autograd: nothing to wait for
            kept = call()
    graph.replay()
    torch.cuda.synchronize()
    first = (lambda o: o[0] if isinstance(o, tuple) else o)
    assert torch.equal(first(kept), first(living).detach())
    del living
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = first(call())
        grads = torch.autograd.grad(out, leaves, grad_outputs=out.detach())
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        eager = first(call())
        want = torch.autograd.grad(eager, leaves, grad_outputs=eager.detach())
        assert torch.equal(out.detach(), eager.detach())
        assert all(torch.equal(a, b) for a, b in zip(grads, want))
        del eager, want
