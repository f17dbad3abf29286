"""Attention for a batch whose sequences share a long prefix.

A serving batch often starts with the same tokens - a system prompt, a document, a few-shot
preamble. Stored once, the prefix's K and V ``[P, Hkv, D]`` are read once per call for all
sequences: the query rows of the whole batch meet them as one matrix product per KV head,
and each sequence's own cache ``[B, T, Hkv, D]`` is read besides. The two parts (and the
splits of each) join by their log-sum-exp. No reference counterpart: the reference decodes
one sequence against its own cache.
"""

from __future__ import annotations

from . import _lib


def shared_prefix_attention(q, k_prefix, v_prefix, k, v, lengths, scale=None, return_lse: bool = False):
    """Dense attention of q's rows over the shared prefix and then over each own cache.

    q [B, Tq, Hq, D]; k_prefix, v_prefix [P, Hkv, D] (P may be 0); k, v [B, T, Hkv, D], of
    which sequence b holds ``lengths[b]`` keys, the call's Tq new tokens among them. Row i of
    sequence b sees every prefix key and the own keys ``j < lengths[b] - Tq + i + 1``; a row
    that sees no key reads as zeros (log-sum-exp -inf). What the caches hold at or past
    ``lengths[b]`` is never used; a key that some row of the call sees must be finite.
    Tensors may be strided views (the head dimension contiguous, rows on 16-byte
    boundaries); others are copied. fp32, fp16 or bf16; D 64 or 128. For 16-bit inputs the
    weights are rounded to the inputs' type for their product with the values (sums, joins and
    log-sum-exp are fp32). ``scale``, positive, defaults to ``D ** -0.5``. Output like q, contiguous; with ``return_lse`` also the natural
    log-sum-exp of every row's scaled logits, fp32 [B, Tq, Hq]."""
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    ops = _lib.torch_ops()
    fn = ops.shared_prefix_attention_lse if return_lse else ops.shared_prefix_attention
    out = fn(q, k_prefix, v_prefix, k, v, lengths, scale)
    _lib.after_call(q.device, "shared_prefix_attention")
    return out
