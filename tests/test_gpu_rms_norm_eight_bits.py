"""rms_norm_quantized: the 8-bit values are those of the float32 quotient of y and the row's scale."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def nearest(quotient, fmt):
    """The format's value nearest to each float32 quotient, ties to even, as float32."""
    most = torch.finfo(fmt).max
    return torch.from_numpy(quotient).clamp(-most, most).to(fmt).float()


@pytest.mark.parametrize("name", ["float8_e4m3fn", "float8_e5m2"])
@pytest.mark.parametrize("width,largest", [(520, 3.7), (2048, 1.0), (4100, 0.0123), (16384, 411.0), (32768, 77.7),
                                           (1000, 3e-36)])
def test_values_are_the_quotients(name, width, largest):
    """x of +-1 has a factor of 1, so that y is the weight, exactly; the scale is the largest one over the
    largest of the format, and a normal float32 number at least.  The weights lie at random, and next to
    the middles between the format's values times the scale, where a quotient that is off by a rounding
    goes to the other side."""
    from gefen_amd import rms_norm_quantized

    fmt = getattr(torch, name)
    most = np.float32(torch.finfo(fmt).max)
    rng = np.random.default_rng(width)
    bits = torch.arange(256, dtype=torch.int16).to(torch.uint8).view(fmt).float()
    values = torch.unique(bits[torch.isfinite(bits) & (bits >= 0)]).numpy()
    middles = (values[1:] + values[:-1]) / 2
    for k in range(8):
        top = np.float32(largest * rng.uniform(0.5, 1.0))
        scale = max(np.float32(top / most), np.float32(2.0 ** -126))
        near = (middles * scale).astype(np.float32)  # and up to three steps of float32 on either side
        near = (near.view(np.int32)[None] + np.arange(-3, 4, dtype=np.int32)[:, None]).reshape(-1).view(np.float32)
        near = near[(near > 0) & (near < top)]
        w = (rng.uniform(-1, 1, width) * top).astype(np.float32)
        at = rng.permutation(width)[:min(near.size, width // 2)]
        w[at] = rng.permutation(near)[:at.size] * rng.choice([-1, 1], at.size).astype(np.float32)
        w[0] = top
        x = torch.from_numpy(rng.choice([-1.0, 1.0], (3, width)).astype(np.float32))
        q, scales = rms_norm_quantized(x.cuda(), torch.from_numpy(w).cuda(), eps=0.0, dtype=fmt)
        assert bool((scales.cpu() == float(scale)).all())
        want = nearest(w / scale, fmt) * x
        assert torch.equal(q.float().cpu(), want), int((q.float().cpu() != want).sum())


@pytest.mark.parametrize("name", ["float8_e4m3fn", "float8_e5m2"])
@pytest.mark.parametrize("largest", [2.0, 1e-36])
def test_zeros_keep_their_sign(name, largest):
    """-0 over a positive scale is -0, beside values that underflow to it."""
    from gefen_amd import rms_norm_quantized

    x = torch.tensor([1.0, -1.0, 0.0, -0.0, 1e-30, -1e-30, 0.0, -0.0, 0.5] * 30, device="cuda")
    w = torch.full_like(x, largest)
    q, _ = rms_norm_quantized(x, w, eps=0.0, dtype=getattr(torch, name))
    assert torch.equal(torch.signbit(q.float()), torch.signbit(x))
