"""rms_norm with dropout in rows of every length, and over the later rows of a workgroup, against the
definition in float64 (bounds: test_gpu_rms_norm), with the generator in whole arrays."""

import numpy as np
import pytest
import torch

from test_gpu_rms_norm import NAMES, SEED, SHAPES, call, definition, kept, make, within

pytestmark = pytest.mark.gpu


def factors(n, p, seed=SEED, offset=0):
    """The same factors as ``kept``, from 64-bit products of 32-bit words."""
    m = np.uint64(0xFFFFFFFF)
    s = np.uint64(32)
    block = np.arange(-(-n // 8), dtype=np.uint64)
    full = lambda v: np.full_like(block, v)  # noqa: E731
    c0, c1, c2, c3 = block & m, block >> s, full(offset & 0xFFFFFFFF), full(offset >> 32)
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):
        a, b = c0 * np.uint64(0xD2511F53), c2 * np.uint64(0xCD9E8D57)
        c0, c1, c2, c3 = (b >> s) ^ c1 ^ np.uint64(k0), b & m, (a >> s) ^ c3 ^ np.uint64(k1), a & m
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = np.stack((c0, c1, c2, c3), 1)
    u = np.stack((words & np.uint64(0xFFFF), words >> np.uint64(16)), 2).reshape(-1)[:n].astype(np.int64)
    cut = round(p * 65536)
    return (torch.from_numpy(u) >= cut).double() * (65536.0 / (65536 - cut))


def compare(dtype, shape, p, offset):
    x, res, w, dy, ds = make(dtype, shape)
    kw = dict(eps=1e-5, dropout=p, seed=SEED, offset=offset)
    got = call(x, res, w, dy, ds, **kw)
    want = definition(dtype, x, res, w, dy, ds, 1e-5, factors(x.numel(), p, offset=offset))
    for a, b, e, name in zip(got, *want, NAMES):
        within(a, b, e, name)
    assert all(torch.equal(a, b) for a, b in zip(got, call(x, res, w, dy, ds, **kw)))


def test_both_generators_agree():
    for n, offset in ((1, 0), (4099, 7), (800, (5 << 32) + 2)):
        assert torch.equal(factors(n, 0.3, offset=offset), kept(n, 0.3, offset=offset))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", [s for s in SHAPES if np.prod(s) > 20000] +
                         [(1, 8200), (1, 16384), (3, 8199), (2, 12001), (2, 16389), (3, 32767), (1, 32768)])
def test_wide_rows(dtype, shape):
    """Rows that a workgroup of 256, 512 and 1024 lanes owns, of whole blocks of eight and not."""
    compare(dtype, shape, 0.3, 7)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", [(9001, 24), (9001, 23), (3000, 1100), (2600, 2051), (2100, 4097), (1100, 8195),
                                   (2100, 8200), (600, 16387)])
def test_many_rows(dtype, shape):
    """More rows than the workgroups of a launch, so that each takes several; odd widths, where eight
    elements take two blocks of the generator."""
    compare(dtype, shape, 0.1, (3 << 32) + 1)
