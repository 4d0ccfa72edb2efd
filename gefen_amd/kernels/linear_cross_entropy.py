"""Softmax cross entropy of an output matrix, with its gradients, without the logits.

    loss = linear_cross_entropy(hidden, lm_head.weight, targets)     # F.cross_entropy(hidden @ W^T, targets)
    loss.backward()

The N x V logits never exist: the library keeps 16 bits per logit of a bounded piece of the
positions at a time (float32 operands: twice as many) and works on positions that have a
loss only.

16-bit gradients, and those of ``reduction`` "none", are formed in backward, so that the
loss's own gradient (a loss scale, a share of a batch) reaches them before they are rounded:
the kept values wait for backward where all positions fit ``workspace_limit`` together.  Where
they do not, bfloat16 gradients of a reduced loss are formed in the forward call and wait in
float32, and float16 ones and those of "none" take the logits' product again.  Float32
operands with "mean" or "sum" have their gradients formed in the forward call (three products
instead of four), and backward multiplies them by the loss's own gradient, which costs nothing
when that is 1.
"""

from __future__ import annotations

from typing import Optional

import torch

from gefen_amd import _lib

__all__ = ["linear_cross_entropy"]

_REDUCTIONS = {"none": _lib.REDUCE_NONE, "mean": _lib.REDUCE_MEAN, "sum": _lib.REDUCE_SUM}


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *,
                         ignore_index: int = -100, label_smoothing: float = 0.0, reduction: str = "mean",
                         workspace_limit: Optional[int] = None) -> torch.Tensor:
    """Cross entropy of the logits ``hidden @ weight.T`` against ``targets``, float32.

    hidden [..., D] and weight [V, D] share a dtype (float32, float16, bfloat16) and may
    have any strides; targets [...] are int64 or int32.  Positions whose target is
    ``ignore_index`` have no loss and no gradient, whatever they hold, and the mean is
    over the others (NaN where there are none, with zero gradients).  A target outside
    [0, V) gives a NaN loss.  No position's loss or gradient depends on what another one
    holds; weight's gradient sums them.  float32 operands are taken in 22 bits, weight's down
    to 2^-28 of its largest element.  ``workspace_limit`` bounds the bytes kept for the gradients
    at a time (4 GiB by default; at least 256 positions are taken at once).  The loss can
    be differentiated once."""
    code = _REDUCTIONS.get(reduction)
    if code is None:
        raise ValueError("Expected reduction to be none, mean or sum, got {!r}".format(reduction))
    label_smoothing = float(label_smoothing)
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError("Expected label_smoothing in [0, 1], got {}".format(label_smoothing))
    limit = 0 if workspace_limit is None else int(workspace_limit)
    if workspace_limit is not None and limit <= 0:
        raise ValueError("Expected a positive workspace_limit, got {}".format(workspace_limit))
    return _lib.host().linear_cross_entropy(hidden, weight, targets, int(ignore_index), label_smoothing, code, limit)
