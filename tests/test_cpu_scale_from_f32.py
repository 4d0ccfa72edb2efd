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


@pytest.mark.parametrize("stage", [16 + 3, 8, 32, 17])
def test_unknown_stages_are_refused(stage):
    more = dict(grad_hidden=FAKE) if stage == 17 else {}  # a forward stage forms no gradients
    assert size(stage=stage, **more) == 0


def test_nothing_to_do():
    assert _lib.load().gefen_scale_from_f32(None, None, 0, None, None, 0, 2, FAKE, None) == _lib.GEFEN_OK


def test_float32_gradients_are_aligned_as_such_and_are_their_own_sum():
    t = task(grad_hidden=FAKE + 2, stage=_lib.LCE_GRADS_F32)
    assert _lib.load().gefen_linear_cross_entropy(ctypes.byref(t), FAKE, 1 << 40, None) == _lib.GEFEN_EINVAL
    k = dict(n=10000, v=4096, grad_weight=FAKE, workspace_limit=1 << 20)
    assert size(**k) - size(stage=_lib.LCE_GRADS_F32, **k) == 4096 * 64 * 4
