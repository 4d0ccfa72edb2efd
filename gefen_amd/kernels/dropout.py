"""Dropout from a counter-based generator: the mask is never stored.

    y = dropout(x, 0.1, seed, offset=layer)               # x kept and scaled by 1 / (1 - p), or zero
    s = dropout(x, 0.1, seed, offset=layer, residual=s)   # added to a residual in the same pass

The mask is a function of ``seed``, ``offset`` and an element's place, so the backward pass
forms it again.  ``seed`` may be an int64 tensor on the device, which the kernels read: a
captured graph takes another mask at each replay when its seed is counted up between them.
Calls of one seed need offsets of their own.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from gefen_amd import _lib

__all__ = ["dropout"]


def probability(p: float, name: str) -> float:
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError("Expected {} in [0, 1], got {}".format(name, p))
    return p


def generator_state(seed: Union[int, torch.Tensor], offset: int) -> Tuple[Optional[torch.Tensor], int, int]:
    """(seed tensor or None, seed as int64, offset) for the host extension."""
    offset = int(offset)
    if not 0 <= offset < 1 << 63:
        raise ValueError("Expected offset in [0, 2^63), got {}".format(offset))
    if isinstance(seed, torch.Tensor):
        return seed, 0, offset
    if isinstance(seed, bool) or not isinstance(seed, int):
        raise TypeError("Expected seed to be an int or an int64 tensor, got {}".format(type(seed).__name__))
    if not -(1 << 63) <= seed < 1 << 64:
        raise ValueError("Expected seed in 64 bits, got {}".format(seed))
    return None, seed - (1 << 64) if seed >= 1 << 63 else seed, offset


def dropout(x: torch.Tensor, p: float, seed: Union[int, torch.Tensor], *, offset: int = 0,
            residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual + x * kept / (1 - p)``, each element of x kept with probability 1 - p (to the
    nearest 2^-16, with which it is also scaled).  x is float32, float16 or bfloat16 of any
    shape and strides, residual of the same shape and dtype.  Element e (in row-major order)
    depends on seed, offset and e only.  A dropped element counts as zero whatever it holds;
    p = 1 drops everything.  The result can be differentiated once."""
    p = probability(p, "p")
    at, value, offset = generator_state(seed, offset)
    return _lib.host().dropout(x, residual, p, at, value, offset)
