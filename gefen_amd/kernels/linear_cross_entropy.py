"""Softmax cross entropy of an output matrix, with its gradients, without the logits.

    loss = linear_cross_entropy(hidden, lm_head.weight, targets)     # F.cross_entropy(hidden @ W^T, targets)
    loss.backward()

The N x V logits never exist: the library keeps 16 bits per logit of a bounded piece of the
positions at a time (float32 ones 22) and works on positions that have a loss only.

With ``reduction`` "mean" or "sum" and bfloat16 or float32 operands the gradients are
formed in the forward call, where the kept values still are (three products instead of
four), and backward multiplies them by the loss's own gradient, which costs nothing when
that is 1.  Float16 gradients are formed in backward, so that a loss scale reaches them
before they are rounded, and so are those of ``reduction`` "none".
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from gefen_amd import _lib

from .gefen_hip import check, device_guard, dtype_code, load_extension, stream_of

__all__ = ["linear_cross_entropy"]

_REDUCTIONS = {"none": _lib.REDUCE_NONE, "mean": _lib.REDUCE_MEAN, "sum": _lib.REDUCE_SUM}


def _check(hidden, weight, targets, label_smoothing, reduction, workspace_limit):
    for name, t in (("hidden", hidden), ("weight", weight), ("targets", targets)):
        if not isinstance(t, torch.Tensor):
            raise TypeError("Expected {} to be a torch.Tensor, got {}".format(name, type(t).__name__))
        if t.device.type != "cuda":
            raise ValueError("Expected {} to be on CUDA, got device {}.".format(name, t.device))
        if t.device != hidden.device:
            raise ValueError("Expected {} on {}, got {}.".format(name, hidden.device, t.device))
    if hidden.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError("Expected hidden to be float32, float16 or bfloat16, got {}".format(hidden.dtype))
    if weight.dtype != hidden.dtype:
        raise ValueError("Expected weight of hidden's dtype {}, got {}".format(hidden.dtype, weight.dtype))
    if targets.dtype not in (torch.int64, torch.int32):
        raise ValueError("Expected targets to be int64 or int32, got {}".format(targets.dtype))
    if weight.dim() != 2:
        raise ValueError("Expected weight to be 2D, got dim={}".format(weight.dim()))
    if hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError("Expected hidden of width {}, got shape {}".format(weight.shape[1], tuple(hidden.shape)))
    if targets.shape != hidden.shape[:-1]:
        raise ValueError("Expected targets of shape {}, got {}".format(tuple(hidden.shape[:-1]),
                                                                       tuple(targets.shape)))
    if weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError("Expected a non-empty weight, got shape {}".format(tuple(weight.shape)))
    if reduction not in _REDUCTIONS:
        raise ValueError("Expected reduction to be none, mean or sum, got {!r}".format(reduction))
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError("Expected label_smoothing in [0, 1], got {}".format(label_smoothing))
    if workspace_limit is not None and workspace_limit <= 0:
        raise ValueError("Expected a positive workspace_limit, got {}".format(workspace_limit))


def _call(hidden, weight, targets, options, losses=None, loss=None, grad_hidden=None, grad_weight=None, grad=None):
    """One library call on 2-D hidden and flat contiguous targets, on the current stream."""
    ignore_index, label_smoothing, reduction, workspace_limit = options
    lib = load_extension()

    def ptr(t: Optional[torch.Tensor]):
        return t.data_ptr() if t is not None else None

    t = _lib.LinearCrossEntropyTask(
        ptr(hidden), ptr(weight), ptr(targets), ptr(losses), ptr(loss), ptr(grad_hidden), ptr(grad_weight), ptr(grad),
        hidden.shape[0], weight.shape[0], weight.shape[1], hidden.stride(0), hidden.stride(1), weight.stride(0),
        weight.stride(1), ignore_index, workspace_limit or 0, label_smoothing, dtype_code(hidden.dtype),
        int(targets.dtype == torch.int32), _REDUCTIONS[reduction], 0)
    nbytes = int(lib.gefen_linear_cross_entropy_workspace_size(ctypes.byref(t)))
    if nbytes == 0:
        check(_lib.GEFEN_EINVAL, "linear_cross_entropy")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=hidden.device)
    check(lib.gefen_linear_cross_entropy(ctypes.byref(t), ws.data_ptr(), nbytes, stream_of(hidden)),
          "linear_cross_entropy")


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, options):
        need_h, need_w = ctx.needs_input_grad[:2]
        h2 = hidden.detach().reshape(-1, hidden.shape[-1])
        w, y = weight.detach(), targets.reshape(-1).contiguous()
        dev = hidden.device
        reduction = options[2]
        with device_guard(hidden):
            ctx.grads = None
            if reduction == "none":
                result = torch.empty(h2.shape[0], dtype=torch.float32, device=dev)
                _call(h2, w, y, options, losses=result)
                result = result.view(targets.shape)
            else:
                result = torch.empty((), dtype=torch.float32, device=dev)
                if (need_h or need_w) and hidden.dtype != torch.float16:
                    ctx.grads = _empty_grads(hidden, weight, need_h, need_w)
                    _call(h2, w, y, options, loss=result, grad_hidden=ctx.grads[0], grad_weight=ctx.grads[1])
                else:
                    _call(h2, w, y, options, loss=result)
        ctx.options = options
        ctx.save_for_backward(hidden, weight, targets)
        return result

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        hidden, weight, targets = ctx.saved_tensors
        need_h, need_w = ctx.needs_input_grad[:2]
        grad = grad.to(torch.float32).reshape(-1).contiguous()
        # the gradients formed in forward are handed over, so a second backward of a
        # retained graph forms them again
        grads, ctx.grads = ctx.grads, None
        with device_guard(hidden):
            if grads is None:
                grads = _empty_grads(hidden, weight, need_h, need_w)
                _call(hidden.detach().reshape(-1, hidden.shape[-1]), weight.detach(), targets.reshape(-1).contiguous(),
                      ctx.options, grad_hidden=grads[0], grad_weight=grads[1], grad=grad)
            else:
                gh, gw = grads
                rc = load_extension().gefen_scale_by(
                    gh.data_ptr() if gh is not None else None, gh.numel() if gh is not None else 0,
                    gw.data_ptr() if gw is not None else None, gw.numel() if gw is not None else 0,
                    dtype_code(hidden.dtype), grad.data_ptr(), stream_of(hidden))
                check(rc, "linear_cross_entropy")
        return grads[0], grads[1], None, None


def _empty_grads(hidden, weight, need_h, need_w):
    return (torch.empty(hidden.shape, dtype=hidden.dtype, device=hidden.device) if need_h else None,
            torch.empty(weight.shape, dtype=weight.dtype, device=weight.device) if need_w else None)


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *,
                         ignore_index: int = -100, label_smoothing: float = 0.0, reduction: str = "mean",
                         workspace_limit: Optional[int] = None) -> torch.Tensor:
    """Cross entropy of the logits ``hidden @ weight.T`` against ``targets``, float32.

    hidden [..., D] and weight [V, D] share a dtype (float32, float16, bfloat16) and may
    have any strides; targets [...] are int64 or int32.  Positions whose target is
    ``ignore_index`` have no loss and no gradient, whatever they hold, and the mean is
    over the others (NaN where there are none, with zero gradients).  A target outside
    [0, V) gives a NaN loss.  ``workspace_limit`` bounds the bytes kept for the gradients
    at a time (4 GiB by default; at least 256 positions are taken at once)."""
    label_smoothing = float(label_smoothing)
    _check(hidden, weight, targets, label_smoothing, reduction, workspace_limit)
    options = (int(ignore_index), label_smoothing, reduction, workspace_limit)
    return _LinearCrossEntropy.apply(hidden, weight, targets, options)
