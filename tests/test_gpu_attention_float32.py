"""float32 attention: the gradients' probabilities are as exact as the output's."""

import pytest
import torch

from test_gpu_attention import attention

pytestmark = pytest.mark.gpu

F = 2.0 ** -24


@pytest.mark.parametrize("d", [64, 96, 127, 128])
def test_small_scores_are_not_lost_beside_a_large_logarithm(d):
    """One query and 64 keys that all score the same small S: P is 1 / 64 and dV is dO / 64.  S is
    a sum of d terms, each a fifth of the spacing of L / scale (L = log 64 + S, L / scale = 22.5 in
    units of base 2: 32.5): added one by one or two by two to a number of that size they are lost, and
    P would be off by d / 5 of those, more than 100 f.  Formed by itself S is exact to d f S, and what
    remains is the rounding of L (6 in base 2: half a spacing is 4 f, and as much of its logarithm), of
    S - L (4 f), all times log 2, exp2 (4 f), the product and the result (2 f): below 32 f."""
    base2 = 1.4426950408889634
    scale = 6.0 / 32.5 / base2
    t = 0.2 * 2.0 ** -18
    g = torch.Generator().manual_seed(d)
    q = torch.ones(1, 1, 1, d).cuda().requires_grad_(True)
    k = torch.full((1, 64, 1, d), t).cuda().requires_grad_(True)
    v = torch.randn(1, 64, 1, d, generator=g).cuda().requires_grad_(True)
    go = torch.randn(1, 1, 1, d, generator=g).cuda()
    dv, = torch.autograd.grad(attention(q, k, v, scale=scale), (v,), grad_outputs=go)
    want = go.double().expand(1, 64, 1, d) / 64
    off = ((dv.double() - want).abs() / want.abs()).max()
    assert float(off) <= 32 * F, float(off) / F


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("queries,keys", [(500, 500), (64, 2000)])
def test_gradients_of_both_sides_are_equally_exact(queries, keys, d):
    """dV against float64: P is off by the roundings of S, of L and of their difference, independent from
    one pair to the next but for L's; relative to the whole that is as in the output, which takes the
    same sums (a factor of 2 covers L, which the output does not need)."""
    g = torch.Generator().manual_seed(d + keys)
    q, k, v, go = (torch.randn(1, n, 4, d, generator=g).cuda() for n in (queries, keys, keys, queries))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = attention(*leaves)
    dv, = torch.autograd.grad(out, (v,), grad_outputs=go)
    p = torch.softmax(torch.einsum("bihd,bjhd->bhij", q.double(), k.double()) * d ** -0.5, -1).detach()
    want = torch.einsum("bhij,bjhd->bihd", p, v.double()).detach(), torch.einsum("bhij,bihd->bjhd", p, go.double())
    err = [float((a.double() - b).norm() / b.norm()) for a, b in zip((out.detach(), dv), want)]
    assert err[1] <= 2 * err[0], err
