"""Root-mean-square norm of a residual stream, with the addition before it.

    y = rms_norm(x, weight)                                   # x / sqrt(mean(x^2) + eps) * weight
    y, s = rms_norm(x, weight, residual=s)                    # s + x, and its norm
    y, s = rms_norm(x, weight, residual=s, dropout=0.1, seed=seed, offset=layer)
    q, scales, s = rms_norm_quantized(x, weight, residual=s)  # y as 8-bit floating point, a scale a row

One pass over a row forward and one backward.  The norm is formed of the sum before that is
rounded to its dtype; the backward pass reads the rounded sum and the norm's factor.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from gefen_amd import _lib
from gefen_amd.kernels.dropout import generator_state, probability

__all__ = ["rms_norm", "rms_norm_quantized"]


def _eps(eps: float) -> float:
    eps = float(eps)
    if not 0.0 <= eps < math.inf:
        raise ValueError("Expected eps to be finite and not negative, got {}".format(eps))
    return eps


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6, residual: Optional[torch.Tensor] = None,
             dropout: float = 0.0, seed: Optional[Union[int, torch.Tensor]] = None,
             offset: int = 0) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """The norm over the last dimension of x [..., width], times weight [width]; with
    ``residual`` (x's shape) that of ``residual + x``, and the sum: (y, s).  One dtype
    (float32, float16, bfloat16), any strides, rows of up to 32768 elements.

    ``dropout`` drops elements of x before the addition, as ``dropout(x, p, seed, offset=offset,
    residual=residual)`` does; it needs a residual and a seed.  The results can be
    differentiated once."""
    eps = _eps(eps)
    dropout = probability(dropout, "dropout")
    at, value, offset = None, 0, int(offset)
    if dropout > 0.0:
        if residual is None or seed is None:
            raise ValueError("Expected a residual and a seed with dropout.")
        at, value, offset = generator_state(seed, offset)
    return _lib.host().rms_norm(x, weight, residual, eps, dropout, at, value, offset)


def rms_norm_quantized(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6,
                       residual: Optional[torch.Tensor] = None,
                       dtype: torch.dtype = torch.float8_e4m3fn) -> Tuple[torch.Tensor, ...]:
    """``rms_norm`` with y in 8 bits: (q, scales), or (q, scales, s) with a residual.  q has the
    dtype ``float8_e4m3fn`` or ``float8_e5m2`` and x's shape, scales [...] are float32, and
    ``q * scales[..., None]`` is y with each row's largest value at the largest of the dtype; q is
    the nearest to the float32 quotient of y and the scale.
    For evaluation: an 8-bit tensor carries no gradient, so it is refused where one is wanted."""
    eps = _eps(eps)
    if dtype not in (torch.float8_e4m3fn, torch.float8_e5m2):
        raise ValueError("Expected dtype to be torch.float8_e4m3fn or torch.float8_e5m2, got {}".format(dtype))
    return _lib.host().rms_norm_quantized(x, weight, residual, eps, dtype == torch.float8_e5m2)
