"""Autograd is told of the parameters that a step writes, as torch's optimizers tell it."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("host", [True, False])
@pytest.mark.parametrize("kind", ["gefen", "muon"])
def test_a_step_counts_as_an_in_place_write(kind, host, monkeypatch):
    """Each way a step runs: the first one, which builds its tables, and those that keep them,
    checked by the host extension or in Python."""
    from gefen_amd import Gefen, GefenMuon, gefen, gefen_muon

    if not host:
        monkeypatch.setattr(gefen, "_gefen_host", None)
        monkeypatch.setattr(gefen_muon, "_gefen_host", None)

    torch.manual_seed(0)
    ps = [torch.nn.Parameter(torch.randn(s, device="cuda").bfloat16()) for s in [(64, 96), (32, 64), (64, 96)]]
    opt = Gefen(ps, lr=1e-3) if kind == "gefen" else GefenMuon(ps, lr=1e-3)
    for _ in range(4):
        for p in ps:
            p.grad = torch.randn_like(p)
        before = [p._version for p in ps]
        h = torch.randn(6, 96, device="cuda").bfloat16().requires_grad_(True)
        product = (h @ ps[0].t()).sum()
        opt.step()
        assert all(p._version > b for p, b in zip(ps, before))
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.backward()


def test_the_kernels_that_update_a_parameter_count_a_version():
    from gefen_amd.kernels import automatic_gefen_fused as fused

    n, period = 64, 16
    p = torch.randn(n, device="cuda")
    grad = torch.randn(n // period, period, device="cuda")
    sign = torch.zeros(n, dtype=torch.uint8, device="cuda")
    magnitude, vmean = torch.zeros(n // period, 1, device="cuda"), torch.ones(n // period, 1, device="cuda")
    codebook = torch.linspace(-1, 1, 256, device="cuda")
    v = p._version
    fused.automatic_gefen_fused_update_cuda(p, grad, sign, magnitude, vmean, codebook, False, 0.9, 1e-3)
    assert p._version > v
    v = p._version
    fused.automatic_gefen_fused_update_from_vmean_cuda(p, grad, sign, magnitude, vmean, codebook, False, 0.9, 1e-3,
                                                       0.1, 0.1, 1e-8)
    assert p._version > v
    v = p._version
    fused.automatic_gefen_period1_update_cuda(p, grad.view(-1), sign, torch.zeros(4, 1, device="cuda"),
                                              torch.ones(n, 1, device="cuda"), codebook, 16, 0.9, 0.99, 1e-3, 0.1, 0.1,
                                              1e-8)
    assert p._version > v


def test_a_step_on_the_output_matrix_is_noticed_by_a_later_backward():
    from gefen_amd import Gefen, linear_cross_entropy

    torch.manual_seed(1)
    w = torch.nn.Parameter(torch.randn(700, 64, device="cuda").bfloat16())
    h = torch.randn(90, 64, device="cuda").bfloat16().requires_grad_(True)
    y = torch.randint(0, 700, (90,), device="cuda")
    opt = Gefen([w], lr=1e-3)
    for _ in range(3):
        loss = linear_cross_entropy(h, w, y, reduction="none")
        w.grad = torch.randn_like(w)
        opt.step()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.sum().backward()
