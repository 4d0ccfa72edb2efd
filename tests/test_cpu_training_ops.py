"""The training operators' C ABI and host logic without a device: argument checks,
workspace sizes, what the wrappers refuse on CPU tensors."""

import ctypes

import numpy as np
import pytest
import torch

from gefen_amd import _lib

FAKE = 1 << 20  # an aligned address that is never read: every call here is refused first


def task(**k):
    t = _lib.LinearCrossEntropyTask()
    t.hidden, t.weight, t.targets, t.loss = FAKE, FAKE, FAKE, FAKE
    t.n, t.v, t.d = 100, 1000, 64
    t.hidden_row_stride = t.weight_row_stride = 64
    t.hidden_col_stride = t.weight_col_stride = 1
    t.ignore_index, t.dtype, t.reduction = -100, _lib.BF16, _lib.REDUCE_MEAN
    for name, value in k.items():
        setattr(t, name, value)
    return t


def size(**k):
    return int(_lib.load().gefen_linear_cross_entropy_workspace_size(ctypes.byref(task(**k))))


def test_struct_mirrors():
    lib = _lib.load()
    assert lib.gefen_struct_size(3) == _lib.GRADIENT_TASK.itemsize
    assert lib.gefen_struct_size(4) == ctypes.sizeof(_lib.LinearCrossEntropyTask)


@pytest.mark.parametrize("bad", [dict(v=0), dict(v=1 << 23), dict(d=0), dict(d=1 << 21), dict(n=-1), dict(n=1 << 31),
                                 dict(dtype=7), dict(label_smoothing=-0.1), dict(label_smoothing=1.5),
                                 dict(label_smoothing=float("nan")), dict(reduction=3), dict(hidden=0), dict(weight=0),
                                 dict(targets=0), dict(hidden=FAKE + 1), dict(weight=FAKE + 1), dict(targets=FAKE + 4),
                                 dict(grad_hidden=FAKE + 1), dict(reduction=_lib.REDUCE_NONE), dict(loss=0),
                                 dict(reduction=_lib.REDUCE_NONE, loss=0, grad_hidden=FAKE)])
def test_linear_cross_entropy_refuses(bad):
    lib = _lib.load()
    t = task(**bad)
    assert lib.gefen_linear_cross_entropy(ctypes.byref(t), FAKE, 1 << 40, None) == _lib.GEFEN_EINVAL
    assert lib.gefen_last_error()


def test_linear_cross_entropy_refuses_a_small_or_missing_workspace():
    lib = _lib.load()
    t = task()
    n = size()
    assert n > 0
    for ws, nbytes in ((FAKE, n - 1), (None, n), (FAKE + 8, n)):
        assert lib.gefen_linear_cross_entropy(ctypes.byref(t), ws, nbytes, None) == _lib.GEFEN_EINVAL
    assert lib.gefen_linear_cross_entropy(None, FAKE, n, None) == _lib.GEFEN_EINVAL
    assert lib.gefen_linear_cross_entropy_workspace_size(None) == 0


def test_workspace_follows_the_limit():
    big = dict(n=65536, v=128256, d=4096, hidden_row_stride=4096, weight_row_stride=4096, grad_hidden=FAKE,
               grad_weight=FAKE)
    fixed = 65536 * 4096 * 2 + 128256 * 4096 * 4 + (256 << 20) + (4 << 20)
    for limit in (256 << 20, 1 << 30, 4 << 30):
        assert size(workspace_limit=limit, **big) <= limit + fixed
    assert size(**big) == size(workspace_limit=4 << 30, **big)
    # a loss alone keeps 12 bytes per 64 logits at most
    big.update(grad_hidden=None, grad_weight=None)
    assert size(**big) <= 65536 * 4096 * 2 + 65536 * 2004 * 12 + (4 << 20)
    # 256 rows at least, whatever the limit
    assert size(workspace_limit=1, n=10000, grad_hidden=FAKE) >= 256 * 1024 * 2
    assert size(n=0) > 0


def rows(*items):
    t = np.zeros(len(items), dtype=_lib.GRADIENT_TASK)
    for r, item in zip(t, items):
        r["src"], r["dst"], r["numel"], r["src_dtype"], r["dst_dtype"] = item
    return t


@pytest.mark.parametrize("item", [(0, FAKE, 5, 0, 0), (FAKE, FAKE, -1, 0, 0), (FAKE, FAKE, 5, 3, 0),
                                  (FAKE + 2, FAKE + 2, 5, 0, 0), (FAKE, FAKE, 1 << 50, 0, 0)])
def test_gradient_norm_refuses(item):
    lib = _lib.load()
    t = rows(item)
    assert lib.gefen_gradient_norm(t.ctypes.data, 1, 2.0, FAKE, FAKE, None) == _lib.GEFEN_EINVAL
    assert lib.gefen_clip_gradients(t.ctypes.data, 1, 2.0, 1.0, FAKE, FAKE, None) == _lib.GEFEN_EINVAL
    assert lib.gefen_scale_gradients(t.ctypes.data, 1, FAKE, 1.0, None) == _lib.GEFEN_EINVAL


def test_clipping_refuses():
    lib = _lib.load()
    ok = rows((FAKE, FAKE, 5, 0, 0))
    other = rows((FAKE, FAKE, 5, 0, 2))
    for call in ((ok, 3.0, 1.0, FAKE, FAKE), (ok, 2.0, -1.0, FAKE, FAKE), (ok, 2.0, float("nan"), FAKE, FAKE),
                 (ok, 2.0, 1.0, None, FAKE), (ok, 2.0, 1.0, FAKE, None), (other, 2.0, 1.0, FAKE, FAKE)):
        t, kind, bound, norm, ws = call
        assert lib.gefen_clip_gradients(t.ctypes.data, 1, kind, bound, norm, ws, None) == _lib.GEFEN_EINVAL
    assert lib.gefen_gradient_norm(ok.ctypes.data, -1, 2.0, FAKE, FAKE, None) == _lib.GEFEN_EINVAL
    assert lib.gefen_gradient_norm(None, 1, 2.0, FAKE, FAKE, None) == _lib.GEFEN_EINVAL
    assert lib.gefen_scale_by(FAKE, 4, None, 4, 0, FAKE, None) == _lib.GEFEN_EINVAL
    assert lib.gefen_scale_by(FAKE, 4, None, 0, 5, FAKE, None) == _lib.GEFEN_EINVAL
    assert lib.gefen_scale_by(FAKE + 1, 4, None, 0, 0, FAKE, None) == _lib.GEFEN_EINVAL
    assert lib.gefen_scale_by(None, 0, None, 0, 0, FAKE, None) == _lib.GEFEN_OK  # nothing to do


def test_norm_workspace_holds_a_partial_per_workgroup():
    lib = _lib.load()
    for sizes in ([1], [0], [16384] * 500, [1 << 33], [5] * 100000):
        t = rows(*[(FAKE, FAKE, n, 0, 0) for n in sizes])
        n = int(lib.gefen_gradient_norm_workspace_size(t.ctypes.data, len(t)))
        assert 8 <= n <= 8 * (8192 + len(t) // 128 + 4)
    assert lib.gefen_gradient_norm_workspace_size(None, 3) == 0


def test_cpu_tensors_and_empty_lists():
    from gefen_amd import clip_grad_norm_, clip_gradients, gradient_norm, linear_cross_entropy

    g = torch.ones(4)
    for call in (lambda: gradient_norm([g]), lambda: clip_gradients([g], 1.0),
                 lambda: linear_cross_entropy(torch.ones(2, 4), torch.ones(3, 4), torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    assert float(gradient_norm([])) == 0.0 and float(clip_gradients([], 1.0)) == 0.0
    p = torch.zeros(3, requires_grad=True)
    assert float(clip_grad_norm_([p], 1.0, error_if_nonfinite=True)) == 0.0


def test_names_are_exported():
    import gefen_amd

    for name in ("linear_cross_entropy", "gradient_norm", "clip_gradients", "clip_grad_norm_"):
        assert name in gefen_amd.__all__ and callable(getattr(gefen_amd, name))


@pytest.mark.parametrize("bad", [dict(stage=3), dict(stage=-1), dict(stage=1, grad_hidden=FAKE), dict(stage=2),
                                 dict(stage=2, grad_hidden=FAKE), dict(stage=2, loss=0),
                                 dict(stage=2, loss=0, losses=FAKE, grad_weight=FAKE),
                                 dict(stage=1, n=10000, workspace_limit=1 << 20),
                                 dict(stage=2, loss=0, grad_weight=FAKE, n=10000, workspace_limit=1 << 20)])
def test_linear_cross_entropy_refuses_stages(bad):
    lib = _lib.load()
    assert size(**bad) == 0
    assert lib.gefen_linear_cross_entropy(ctypes.byref(task(**bad)), FAKE, 1 << 40, None) == _lib.GEFEN_EINVAL


def test_a_backward_stage_fits_the_workspace_of_its_forward_stage():
    for n, v, d in ((1, 1, 1), (48, 1000, 96), (300, 50257, 768), (2000, 32003, 1001)):
        for dtype in (_lib.F32, _lib.F16, _lib.BF16):
            for reduction in (_lib.REDUCE_NONE, _lib.REDUCE_MEAN):
                k = dict(n=n, v=v, d=d, dtype=dtype, reduction=reduction)
                loss = 0 if reduction == _lib.REDUCE_NONE else FAKE
                forward = size(stage=1, loss=loss, **k)
                for g in (dict(grad_hidden=FAKE), dict(grad_weight=FAKE), dict(grad_hidden=FAKE, grad_weight=FAKE)):
                    assert 0 < size(stage=2, loss=0, **k, **g) <= forward
