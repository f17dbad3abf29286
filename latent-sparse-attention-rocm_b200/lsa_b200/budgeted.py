"""Decoding under a shared prefix with every sequence's own cache held to a budget.

The loop that ``shared_prefix_attention``, ``scored_attention`` and ``evict`` are for: a batch
starts from one long prompt, stored once; each sequence appends its tokens to its own cache,
every step scores the cached keys by the attention they receive, and when the room is used up
the keys that matter least leave. No reference counterpart.

    cache = BudgetedCache(k, v, lengths, budget=2048, room=64, k_prefix=kp, v_prefix=vp)
    for q, k_new, v_new in steps:              # [B, Tq, Hq, D], [B, Tq, Hkv, D] twice
        out = cache.step(q, k_new, v_new)
"""

from __future__ import annotations

import math

import torch

from .eviction import EvictedCache, evict, scored_attention


class BudgetedCache:
    """The own caches of a decoding batch: at most ``budget`` keys a (sequence, KV head) after an
    eviction, ``room`` more until the next.

    k, v [B, T, Hkv, D] hold the sequences' own prompts, ``lengths`` [B] (host integers) how much of
    them; ``scores`` fp32 [B, Hkv, T] what they have collected so far (zeros when None: then
    an eviction keeps the oldest of the keys that nothing has read). The sinks and the window
    are those of ``evict``."""

    def __init__(self, k, v, lengths, budget: int, room: int, window_size: int = 64, sink_size: int = 4,
                 k_prefix=None, v_prefix=None, scores=None):
        if room < 1:
            raise ValueError(f"a budgeted cache needs room to append to, got {room}")
        B, T, Hkv, _ = k.shape
        lengths = [int(n) for n in lengths]
        if len(lengths) != B or any(n < 0 or n > T for n in lengths):
            raise ValueError(f"one length in [0, {T}] a sequence, got {lengths}")
        self.budget, self.capacity = int(budget), int(budget) + int(room)
        self.window_size, self.sink_size = window_size, sink_size
        self.k_prefix, self.v_prefix = k_prefix, v_prefix
        if scores is None:
            scores = torch.zeros(B, Hkv, T, dtype=torch.float32, device=k.device)
        self.k, self.v, self.scores = k, v, scores
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=k.device)
        self._longest = max(lengths, default=0)  # of the batch, known without asking the device
        self._rows = torch.arange(B, device=k.device)[:, None]
        self._take(self._evicted(), min(self._longest, self.budget))

    def _evicted(self):
        return evict(self.k, self.v, self.scores, self.lengths, self.budget, self.window_size, self.sink_size,
                     self.capacity)

    def _take(self, cache, longest):
        self.k, self.v, self.scores, self.lengths = cache.k, cache.v, cache.scores, cache.lengths
        self._longest = longest

    def _check_step(self, q, k_new, v_new, scale):
        """ValueError for a step that the writes below would spread over other slots (an indexed write
        repeats what has one entry) or that the operator would refuse once they are done."""
        B, _, Hkv, D = self.k.shape
        if q.dim() != 4 or q.shape[0] != B or q.shape[3] != D or q.shape[2] % Hkv or q.shape[2] < Hkv:
            raise ValueError(f"a step's q is [{B}, Tq, Hq, {D}], Hq a multiple of {Hkv}, got {list(q.shape)}")
        want = (B, q.shape[1], Hkv, D)
        if k_new.shape != want or v_new.shape != want:
            raise ValueError(f"a step's keys and values are {list(want)}, got {list(k_new.shape)}, {list(v_new.shape)}")
        if any(t.dtype != self.k.dtype or t.device != self.k.device for t in (q, k_new, v_new)):
            raise ValueError(f"a step's tensors are {self.k.dtype} on {self.k.device}, as the cache")
        if scale is not None and not 0.0 < scale < math.inf:
            raise ValueError(f"the scale must be positive, got {scale}")
        if q.shape[1] > self.capacity - self.budget:
            raise ValueError(f"a step of {q.shape[1]} tokens does not fit the room of {self.capacity - self.budget}")

    def step(self, q, k_new, v_new, scale=None):
        """Append the step's Tq tokens, attend to the prefix and the own cache, score the keys.
        Evicts first when the longest sequence has no room for them. q [B, Tq, Hq, D], k_new and
        v_new [B, Tq, Hkv, D]; a refused step (ValueError) leaves the cache as it was. Output like q."""
        self._check_step(q, k_new, v_new, scale)
        Tq, cache, longest = q.shape[1], self, self._longest
        if longest + Tq > self.capacity:
            cache, longest = self._evicted(), min(longest, self.budget)
        at = cache.lengths.long()[:, None] + torch.arange(Tq, device=q.device)
        cache.k[self._rows, at], cache.v[self._rows, at] = k_new, v_new  # past the lengths: not yet the cache's
        lengths = cache.lengths + Tq
        out, scores = scored_attention(q, cache.k, cache.v, lengths, cache.scores, scale, self.k_prefix,
                                       self.v_prefix)
        self._take(EvictedCache(cache.k, cache.v, scores, lengths, None), longest + Tq)
        return out
