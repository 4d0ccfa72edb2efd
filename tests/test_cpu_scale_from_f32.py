"""gefen_scale_from_f32 and float32 gradients of a 16-bit task: argument checks without a device."""

import ctypes

import pytest

from gefen_amd import _lib
from test_cpu_training_ops import FAKE, size, task


@pytest.mark.parametrize("a", [(FAKE, FAKE, 4, None, FAKE, 4, 0, FAKE), (FAKE, None, 4, None, None, 0, 1, FAKE),
                               (FAKE, FAKE, -1, None, None, 0, 1, FAKE), (FAKE, FAKE, 4, None, None, 0, 9, FAKE),
                               (FAKE + 2, FAKE, 4, None, None, 0, 2, FAKE), (FAKE, FAKE + 1, 4, None, None, 0, 2, FAKE),
                               (FAKE, FAKE + 2, 4, None, None, 0, 0, FAKE), (FAKE, FAKE, 4, None, None, 0, 2, None)])
def test_refusals(a):
    assert _lib.load().gefen_scale_from_f32(*a, None) == _lib.GEFEN_EINVAL


def test_nothing_to_do():
    assert _lib.load().gefen_scale_from_f32(None, None, 0, None, None, 0, 2, FAKE, None) == _lib.GEFEN_OK


def test_float32_gradients_are_aligned_as_such_and_are_their_own_sum():
    t = task(grad_hidden=FAKE + 2, grads_f32=1)
    assert _lib.load().gefen_linear_cross_entropy(ctypes.byref(t), FAKE, 1 << 40, None) == _lib.GEFEN_EINVAL
    k = dict(n=10000, v=4096, grad_weight=FAKE, workspace_limit=1 << 20)
    assert size(**k) - size(grads_f32=1, **k) == 4096 * 64 * 4
