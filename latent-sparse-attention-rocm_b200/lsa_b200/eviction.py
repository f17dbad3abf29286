"""A cache held to a budget: attention that scores the keys, and the eviction of the lowest.

``scored_attention`` is ``shared_prefix_attention`` that also adds, to a running score per
own key and KV head, the attention weight the key received from every row and query head of
the call. ``evict`` brings every (sequence, KV head) back to ``budget`` keys: the first
``sink_size`` and the last ``window_size`` stay, as the selection's sinks and window do, and
of the others those with the highest score. Kept keys keep their order, so an evicted cache
is a cache like any other: attended, scored, appended to, indexed. No reference counterpart.

    out, scores = scored_attention(q, k, v, lengths, scores)      # every step
    cache = evict(k, v, scores, lengths, budget, capacity=room)   # when the room runs out
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib


class EvictedCache(NamedTuple):
    k: torch.Tensor  # [B, capacity, Hkv, D]; zeros past the kept keys
    v: torch.Tensor  # [B, capacity, Hkv, D]
    scores: torch.Tensor  # fp32 [B, Hkv, capacity]; zeros past the kept keys
    lengths: torch.Tensor  # int32 [B]
    ids: torch.Tensor  # int32 [B, Hkv, capacity]: kept keys' indices in the old cache, ascending; -1 past them


def scored_attention(q, k, v, lengths, scores, scale=None, k_prefix=None, v_prefix=None):
    """(output, scores): attention over the own caches, after a shared prefix when one is given,
    and the scores with this call's weights added.

    Arguments as ``shared_prefix_attention``; scores fp32 [B, Hkv, T] (zero for a new key).
    scores_out[b, h, j] = scores[b, h, j] + the sum of key j's weights over the call's rows
    that see it and the query heads of KV head h, the weights those of the whole softmax
    (prefix keys included); entries at or past ``lengths[b]`` are copied. The prefix's own keys
    are not scored. Every entry has one writer: the same inputs give the same bits."""
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    out = _lib.torch_ops().scored_attention(q, k, v, lengths, scores, scale, k_prefix, v_prefix)
    _lib.after_call(q.device, "scored_attention")
    return out


def evict(k, v, scores, lengths, budget: int, window_size: int = 64, sink_size: int = 4, capacity=None):
    """Keep at most ``budget`` keys of every (sequence, KV head); returns an ``EvictedCache``.

    k, v [B, T, Hkv, D] (any dtype whose rows are a multiple of 16 bytes), scores fp32
    [B, Hkv, T], lengths [B]. With n = lengths[b] <= budget every key stays. Else the first
    ``sink_size``, the last ``window_size`` and the highest-scored others stay: scores in the
    order of the selection's packed keys (+NaN above +inf, -0 below +0), ties to the lower
    index. The new cache has ``capacity`` slots (default ``budget``), zero past the kept keys."""
    capacity = budget if capacity is None else capacity
    r = _lib.torch_ops().evict(k, v, scores, lengths, budget, window_size, sink_size, capacity)
    _lib.after_call(k.device, "evict")
    return EvictedCache(*r)
