"""Softmax attention with its gradients, without the probabilities.

    out = attention(query, key, value, causal=True)      # softmax(query @ key^T / sqrt(width)) @ value
    out.backward(...)

One pass over the keys with a running maximum and sum; the backward pass forms the
probabilities again from the logarithm of each row's sum, in one kernel that owns queries
and one that owns keys, so that no sum depends on scheduling.  Heads that share a key head
are rows of one problem.
"""

from __future__ import annotations

from typing import Optional

import torch

from gefen_amd import _lib

__all__ = ["attention"]


def attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, *, causal: bool = False,
              scale: Optional[float] = None, key_lengths: Optional[torch.Tensor] = None,
              offsets: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of query [batch, queries, heads, width] over key and value [batch, keys,
    kv_heads, width], of one dtype (float32, float16, bfloat16), any strides, a width of up to
    128; ``heads`` is a multiple of ``kv_heads`` and head h reads key head
    ``h // (heads // kv_heads)``.  ``scale`` (1 / sqrt(width) by default) is not negative.

    Query i sees key j where ``j < key_lengths[b]`` (int32 or int64 [batch] on the device) and,
    with ``causal``, where ``j <= i + keys - queries``: the last query at the last key (of the
    tensor, not of ``key_lengths``).  With
    ``offsets`` (int32 or int64 [sequences + 1] on the device, ascending) the tensors are packed
    sequences [tokens, heads, width], sequence s holding the tokens from ``offsets[s]`` to
    ``offsets[s + 1]``, and a token sees its own sequence only.

    A query that sees no key gives zeros and has no gradient, and so does a key that no query
    sees; what is not seen does not reach a result, whatever it holds.  The result can be
    differentiated once.  ``batch * kv_heads`` times the blocks of 128 keys, or of 128 of
    ``queries * heads / kv_heads``, is below 2^24."""
    if scale is not None:
        scale = float(scale)
        if not 0.0 <= scale < float("inf"):
            raise ValueError("Expected scale to be finite and not negative, got {}".format(scale))
    return _lib.host().attention(query, key, value, key_lengths, offsets, bool(causal), scale)
