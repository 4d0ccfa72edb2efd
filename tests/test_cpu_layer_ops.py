"""The layer operators' C ABI and host logic without a device: argument checks, workspace
sizes, what the wrappers refuse on CPU tensors."""

import ctypes

import pytest
import torch

from gefen_amd import _lib

FAKE = 1 << 20  # an aligned address that is never read: every call here is refused first


def attention_task(**k):
    t = _lib.AttentionTask()
    for name in ("query", "key", "value", "out", "lse", "grad_out", "grad_query", "grad_key", "grad_value"):
        setattr(t, name, FAKE)
    t.batch, t.queries, t.keys, t.heads, t.kv_heads, t.width = 2, 100, 120, 8, 2, 64
    t.scale, t.dtype = 0.125, _lib.BF16
    for name, value in k.items():
        setattr(t, name, value)
    return t


def rms_task(**k):
    t = _lib.RmsNormTask()
    for name in ("x", "weight", "y", "rstd", "grad_y", "grad_x", "grad_weight"):
        setattr(t, name, FAKE)
    t.rows, t.width, t.x_row_stride, t.grad_y_row_stride, t.eps, t.dtype = 100, 64, 64, 64, 1e-6, _lib.BF16
    for name, value in k.items():
        setattr(t, name, value)
    return t


def test_struct_mirrors():
    lib = _lib.load()
    assert lib.gefen_struct_size(5) == ctypes.sizeof(_lib.AttentionTask)
    assert lib.gefen_struct_size(6) == ctypes.sizeof(_lib.RmsNormTask)


@pytest.mark.parametrize("bad", [dict(dtype=7), dict(batch=-1), dict(queries=-1), dict(keys=-1), dict(heads=0),
                                 dict(kv_heads=0), dict(kv_heads=3), dict(width=0), dict(width=129),
                                 dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
                                 dict(queries=1 << 31), dict(keys=1 << 31), dict(batch=1 << 31),
                                 dict(queries=1 << 29), dict(batch=1 << 28), dict(heads=1 << 20),
                                 dict(query=0), dict(key=0), dict(value=0), dict(out=0), dict(query=FAKE + 1),
                                 dict(key=FAKE + 1), dict(lse=FAKE + 2), dict(key_lengths=FAKE + 2),
                                 dict(key_lengths=FAKE + 4, lengths_int64=1), dict(offsets=FAKE),
                                 dict(offsets=FAKE, batch=1), dict(offsets=FAKE + 1, batch=1, keys=100),
                                 dict(offsets=FAKE, batch=1, keys=100, sequences=-1),
                                 dict(offsets=FAKE, batch=1, keys=100, key_lengths=FAKE)])
def test_attention_refuses(bad):
    lib = _lib.load()
    t = attention_task(**bad)
    assert lib.gefen_attention_forward(ctypes.byref(t), FAKE, 1 << 40, None) == _lib.GEFEN_EINVAL
    assert lib.gefen_last_error()
    assert lib.gefen_attention_backward(ctypes.byref(t), FAKE, 1 << 40, None) == _lib.GEFEN_EINVAL


def test_attention_backward_refuses():
    lib = _lib.load()
    t = attention_task()
    n = int(lib.gefen_attention_backward_workspace_size(ctypes.byref(t)))
    assert n >= 2 * 100 * 8 * 4
    for ws, size in ((FAKE, n - 1), (None, n), (FAKE + 8, n)):
        assert lib.gefen_attention_backward(ctypes.byref(t), ws, size, None) == _lib.GEFEN_EINVAL
    for bad in (dict(lse=0), dict(grad_out=0), dict(grad_query=0), dict(grad_key=0), dict(grad_value=0),
                dict(grad_key=FAKE + 1)):
        assert lib.gefen_attention_backward(ctypes.byref(attention_task(**bad)), FAKE, n, None) == _lib.GEFEN_EINVAL
    assert lib.gefen_attention_forward(None, FAKE, 1 << 40, None) == _lib.GEFEN_EINVAL
    assert lib.gefen_attention_backward(None, FAKE, n, None) == _lib.GEFEN_EINVAL
    assert lib.gefen_attention_backward_workspace_size(None) == 0
    assert lib.gefen_attention_forward_workspace_size(None) == 0
    # few rows over many keys are split, and their parts need a workspace
    t = attention_task(queries=1, keys=8192)
    n = int(lib.gefen_attention_forward_workspace_size(ctypes.byref(t)))
    assert n >= 2 * 2 * 8 * 64 * 4
    for ws, size in ((FAKE, n - 1), (None, n), (FAKE + 8, n)):
        assert lib.gefen_attention_forward(ctypes.byref(t), ws, size, None) == _lib.GEFEN_EINVAL
    # nothing to do
    assert lib.gefen_attention_forward(ctypes.byref(attention_task(batch=0)), None, 0, None) == _lib.GEFEN_OK
    assert lib.gefen_attention_backward(ctypes.byref(attention_task(batch=0)), FAKE, 1 << 20, None) == _lib.GEFEN_OK


@pytest.mark.parametrize("bad", [dict(dtype=-1), dict(rows=-1), dict(rows=1 << 40), dict(width=0), dict(width=32769),
                                 dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(dropout=-0.1),
                                 dict(dropout=1.1), dict(dropout=float("nan")), dict(seed_at=FAKE + 4), dict(x=0),
                                 dict(weight=0), dict(x=FAKE + 1), dict(weight=FAKE + 1), dict(rstd=FAKE + 2)])
def test_rms_norm_refuses(bad):
    lib = _lib.load()
    t = rms_task(**bad)
    assert lib.gefen_rms_norm_forward(ctypes.byref(t), None) == _lib.GEFEN_EINVAL
    assert lib.gefen_last_error()
    assert lib.gefen_rms_norm_backward(ctypes.byref(t), FAKE, 1 << 40, None) == _lib.GEFEN_EINVAL


def test_rms_norm_refuses_by_direction():
    lib = _lib.load()
    for bad in (dict(y=0), dict(y=FAKE + 1), dict(residual=FAKE + 1), dict(sum=FAKE + 1), dict(out=3), dict(out=-1),
                dict(out=_lib.RMS_E4M3), dict(out=_lib.RMS_E5M2, scales=FAKE + 1)):
        assert lib.gefen_rms_norm_forward(ctypes.byref(rms_task(**bad)), None) == _lib.GEFEN_EINVAL
    t = rms_task()
    n = int(lib.gefen_rms_norm_backward_workspace_size(ctypes.byref(t)))
    assert n >= 64 * 4
    for ws, size in ((FAKE, n - 1), (None, n), (FAKE + 4, n)):
        assert lib.gefen_rms_norm_backward(ctypes.byref(t), ws, size, None) == _lib.GEFEN_EINVAL
    for bad in (dict(rstd=0), dict(grad_y=0), dict(grad_y=FAKE + 1), dict(grad_sum=FAKE + 1), dict(grad_x=FAKE + 1),
                dict(grad_residual=FAKE + 1), dict(grad_weight=FAKE + 1)):
        assert lib.gefen_rms_norm_backward(ctypes.byref(rms_task(**bad)), FAKE, n, None) == _lib.GEFEN_EINVAL
    assert lib.gefen_rms_norm_forward(None, None) == _lib.GEFEN_EINVAL
    assert lib.gefen_rms_norm_backward(None, FAKE, n, None) == _lib.GEFEN_EINVAL
    assert lib.gefen_rms_norm_backward_workspace_size(None) == 0
    assert lib.gefen_rms_norm_forward(ctypes.byref(rms_task(rows=0)), None) == _lib.GEFEN_OK


def test_dropout_refuses():
    lib = _lib.load()
    for x, r, y, n, dt, p, seed_at in ((FAKE, None, FAKE, 8, 5, 0.1, None), (FAKE, None, FAKE, -1, 0, 0.1, None),
                                       (FAKE, None, FAKE, 1 << 48, 0, 0.1, None), (FAKE, None, FAKE, 8, 0, -0.1, None),
                                       (FAKE, None, FAKE, 8, 0, 1.5, None), (FAKE, None, FAKE, 8, 0, float("nan"), None),
                                       (None, None, FAKE, 8, 0, 0.1, None), (FAKE, None, None, 8, 0, 0.1, None),
                                       (FAKE + 2, None, FAKE, 8, 0, 0.1, None), (FAKE, FAKE + 1, FAKE, 8, 2, 0.1, None),
                                       (FAKE, None, FAKE + 1, 8, 1, 0.1, None), (FAKE, None, FAKE, 8, 0, 0.1, FAKE + 4)):
        assert lib.gefen_dropout(x, r, y, n, dt, p, seed_at, 0, 0, None) == _lib.GEFEN_EINVAL
        assert lib.gefen_last_error()
    assert lib.gefen_dropout(None, None, None, 0, 0, 0.1, None, 0, 0, None) == _lib.GEFEN_OK


def test_names_are_exported():
    import gefen_amd

    for name in ("attention", "rms_norm", "rms_norm_quantized", "dropout"):
        assert name in gefen_amd.__all__ and callable(getattr(gefen_amd, name))


def test_cpu_tensors_are_refused():
    from gefen_amd import attention, dropout, rms_norm, rms_norm_quantized

    x, q = torch.ones(4, 8), torch.ones(1, 2, 2, 8)
    for call in (lambda: attention(q, q, q), lambda: rms_norm(x, x[0]), lambda: rms_norm(x, x[0], residual=x),
                 lambda: rms_norm_quantized(x, x[0]), lambda: dropout(x, 0.1, 3)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_arguments_that_no_device_is_needed_for():
    from gefen_amd import attention, dropout, rms_norm, rms_norm_quantized

    x, q = torch.ones(4, 8), torch.ones(1, 2, 2, 8)
    for call in (lambda: attention(q, q, q, scale=-1.0), lambda: attention(q, q, q, scale=float("nan")),
                 lambda: rms_norm(x, x[0], eps=-1.0), lambda: rms_norm(x, x[0], dropout=2.0),
                 lambda: rms_norm(x, x[0], dropout=0.1, seed=1), lambda: rms_norm(x, x[0], residual=x, dropout=0.1),
                 lambda: rms_norm_quantized(x, x[0], dtype=torch.float16), lambda: dropout(x, 1.1, 1),
                 lambda: dropout(x, 0.1, 1 << 64), lambda: dropout(x, 0.1, 1, offset=-1)):
        with pytest.raises(ValueError, match="Expected"):
            call()
    for call in (lambda: dropout(x, 0.1, "1"), lambda: dropout(x, 0.1, 1.0), lambda: attention(q, q, None),
                 lambda: rms_norm(x, None)):
        with pytest.raises(TypeError):
            call()
