"""Global gradient norm and clipping, between ``loss.backward()`` and ``opt.step()``.

    t = (sum |g|^2)^(1/2)  (or sum |g|, max |g|),   g <- g * min(1, max_norm / (t + 1e-6))

``clip_grad_norm_`` takes parameters as ``torch.nn.utils.clip_grad_norm_`` does;
``gradient_norm`` and ``clip_gradients`` take the gradients themselves, any mixture of
float32, float16 and bfloat16 on one device.  The norm is a 0-d float32 tensor on that
device and nothing waits for it: one or two launches for the norm and as many for the
scaling (128 tensors each), no synchronisation.  Its sums are float64, so the result
does not depend on scheduling, and neither large nor small gradients leave the range.
"""

from __future__ import annotations

import math
from typing import Iterable, List, Optional, Sequence, Union

import torch

from gefen_amd import _lib

__all__ = ["gradient_norm", "clip_gradients", "clip_grad_norm_"]


def _norm_type(norm_type: float) -> float:
    norm_type = float(norm_type)
    if norm_type not in (1.0, 2.0, math.inf):
        raise ValueError("Expected norm_type to be 1, 2 or inf, got {}".format(norm_type))
    return norm_type


def _bound(max_norm: float) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError("Expected max_norm to be non-negative, got {}".format(max_norm))
    return max_norm


def _as_list(tensors, name: str) -> List[torch.Tensor]:
    if isinstance(tensors, torch.Tensor):
        return [tensors]
    if not isinstance(tensors, (list, tuple)):
        raise TypeError("Expected {} to be a list of tensors, got {}".format(name, type(tensors).__name__))
    return list(tensors)


def _dense(grads: List[torch.Tensor], out: Optional[List[torch.Tensor]] = None):
    """Contiguous stand-ins for tensors that are not one dense run of elements, or stand for
    the negative of their memory, and the (destination, stand-in) pairs to copy back."""
    src, dst, back = list(grads), list(grads if out is None else out), []
    for k, (g, o) in enumerate(zip(grads, dst)):
        if not (g.is_contiguous() and o.is_contiguous()) or g.is_neg() or o.is_neg():
            src[k], dst[k] = g.resolve_neg().contiguous(), torch.empty(g.shape, dtype=o.dtype, device=g.device)
            back.append((o, dst[k]))
    return src, dst, back


def gradient_norm(gradients: Sequence[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The norm over every element of all gradients: a 0-d float32 tensor on their device
    (zero on the CPU for an empty list).  A sharded model joins its shards' norms itself
    (for 2: the root of the all-reduced sum of squares) and passes the result to
    ``clip_gradients(..., total_norm=...)``."""
    norm_type = _norm_type(norm_type)
    grads = _as_list(gradients, "gradients")
    if not grads:
        return torch.zeros(())
    host = _lib.host()
    norm = host.gradient_norm(grads, norm_type)
    return norm if norm is not None else host.gradient_norm(_dense(grads)[0], norm_type)


def clip_gradients(gradients: Sequence[torch.Tensor], max_norm: float, norm_type: float = 2.0, *,
                   out: Optional[Sequence[torch.Tensor]] = None,
                   total_norm: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Scale the gradients to a norm of at most ``max_norm`` and return the norm they had.

    In place without ``out`` (and then not written at all where the norm is within the
    bound); else ``out[i]``, of the same shape and any of the three dtypes, receives the
    scaled ``gradients[i]``, rounded once: float32 accumulators into bfloat16 gradients
    in one pass.  ``total_norm`` (0-d float32, same device) replaces the norm of these
    gradients where they are only a part of the model's.  A NaN norm makes every
    gradient NaN, an infinite one makes them zero (and NaN where infinite)."""
    norm_type, max_norm = _norm_type(norm_type), _bound(max_norm)
    grads = _as_list(gradients, "gradients")
    outs = None if out is None else _as_list(out, "out")
    if total_norm is not None:
        if not isinstance(total_norm, torch.Tensor):
            raise TypeError("Expected total_norm to be a torch.Tensor, got {}".format(type(total_norm).__name__))
        if total_norm.dim() != 0 or total_norm.dtype != torch.float32:
            raise ValueError("Expected total_norm to be a 0-d float32 tensor.")
        if grads and total_norm.device != grads[0].device:
            raise ValueError("Expected total_norm on the gradients' device, got {}.".format(total_norm.device))
    if not grads:
        if outs:
            raise ValueError("Expected as many output tensors as gradients.")
        return torch.zeros(()) if total_norm is None else total_norm
    host = _lib.host()
    norm = host.clip_gradients(grads, outs, max_norm, norm_type, total_norm)
    if norm is None:
        with torch.no_grad():
            src, dst, back = _dense(grads, outs)
            norm = host.clip_gradients(src, dst, max_norm, norm_type, total_norm)
            for o, t in back:
                o.copy_(t)
    return norm


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float,
                    norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Clip the gradients of ``parameters`` in place to a global norm of at most
    ``max_norm``; returns the norm before.  Parameters without a gradient are skipped.
    ``error_if_nonfinite`` waits for the norm and raises before anything is written."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if error_if_nonfinite and grads:
        total = gradient_norm(grads, norm_type)
        if not bool(torch.isfinite(total)):
            raise RuntimeError("The norm of order {} of the gradients is non-finite, so they cannot be clipped."
                               .format(float(norm_type)))
        return clip_gradients(grads, max_norm, norm_type, total_norm=total)
    return clip_gradients(grads, max_norm, norm_type)
