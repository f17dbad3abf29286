"""Cases of the shared-prefix attention, the scored attention and the cache eviction.

The three operators of a serving loop whose sequences start with the same long prompt and
whose own caches are held to a budget: attention over a prefix stored once and over each
sequence's own cache; the same attention that also adds every own key's attention weight to a
running score; the eviction of the keys whose score is lowest.

``own`` false: the plain forms, elementary torch operations in fp32. ``own`` true: the calls a
user makes of ``lsa_b200``.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases


def listed():
    return [
        # --- attention over a shared prefix
        # a few requests under a short system prompt: the latency of one decode step
        {"name": "prefix_decode_small", "op": "prefix", "B": 4, "Tq": 1, "Hq": 32, "Hkv": 8, "D": 128, "P": 2048,
         "T": 256, "dtype": "bf16"},
        # a full decode batch under a 32k document, ragged own caches
        {"name": "prefix_decode_64x32k", "op": "prefix", "B": 64, "Tq": 1, "Hq": 32, "Hkv": 8, "D": 128, "P": 32768,
         "T": 1024, "dtype": "bf16"},
        # 128k of shared context, 8 query heads per KV head
        {"name": "prefix_decode_16x128k", "op": "prefix", "B": 16, "Tq": 1, "Hq": 64, "Hkv": 8, "D": 128,
         "P": 131072, "T": 2048, "dtype": "fp16"},
        # the requests' own prompts, 64 tokens each, after an odd prefix: the compute-bound end
        {"name": "prefix_chunk_32x64", "op": "prefix", "B": 32, "Tq": 64, "Hq": 32, "Hkv": 8, "D": 128, "P": 10007,
         "T": 577, "dtype": "bf16"},
        # a small model's heads, five tokens verified per step
        {"name": "prefix_verify_d64", "op": "prefix", "B": 24, "Tq": 5, "Hq": 8, "Hkv": 2, "D": 64, "P": 16001,
         "T": 777, "dtype": "fp16"},
        # --- attention that scores the cache
        # one sequence's decode step, 32k of cache
        {"name": "scored_decode_1x32k", "op": "scored", "B": 1, "Tq": 1, "Hq": 32, "Hkv": 8, "D": 128, "P": 0,
         "T": 32768, "dtype": "bf16"},
        # a decode batch on budgeted caches under a shared prompt
        {"name": "scored_decode_48x8k", "op": "scored", "B": 48, "Tq": 1, "Hq": 32, "Hkv": 8, "D": 128, "P": 4096,
         "T": 8191, "dtype": "bf16"},
        # the last 32 rows of a prompt score its keys before the prompt is compressed
        {"name": "scored_window_4x32k", "op": "scored", "B": 4, "Tq": 32, "Hq": 32, "Hkv": 8, "D": 128, "P": 0,
         "T": 32768, "dtype": "bf16"},
        # --- eviction
        # a cache that has grown 64 tokens past its budget
        {"name": "evict_step_1x2112", "op": "evict", "B": 1, "Hkv": 8, "D": 128, "T": 2112, "ragged": False,
         "budget": 2048, "window": 64, "sink": 4, "dtype": "bf16"},
        # a ragged batch back to its budget
        {"name": "evict_batch_64x8k", "op": "evict", "B": 64, "Hkv": 8, "D": 128, "T": 8191, "ragged": True,
         "budget": 2048, "window": 64, "sink": 4, "dtype": "bf16"},
        # long prompts compressed after their prefill
        {"name": "evict_prompt_4x128k", "op": "evict", "B": 4, "Hkv": 8, "D": 128, "T": 131072, "ragged": False,
         "budget": 8192, "window": 256, "sink": 4, "dtype": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["prefix", "prefix", "scored", "scored", "evict"])
    Hkv, D = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "evict":
        B, T = _log(rng, 1, 64), _log(rng, 64, 131072)
        B = max(1, min(B, 64 * 8192 // T))
        budget = max(1, min(T, int(T * rng.uniform(0.05, 1.0))))
        window = min(rng.choice([1, 16, 64, 256]), budget // 2)
        sink = min(rng.choice([0, 1, 4]), budget - window)
        return {"op": op, "B": B, "Hkv": Hkv, "D": D, "T": T, "ragged": rng.random() < 0.5, "budget": budget,
                "window": window, "sink": sink, "dtype": dtype}
    Hq = Hkv * rng.choice([1, 2, 3, 4, 4, 6, 8, 8])
    Tq = rng.choice([1, 1, 1, 2, 3, 5, 8, 16, 32, 61])
    if op == "prefix":
        B, P = _log(rng, 1, 128), _log(rng, 128, 131072)
        T = max(Tq, _log(rng, 1, 4096))
    else:
        B, T = _log(rng, 1, 64), max(Tq, _log(rng, 64, 131072))
        P = rng.choice([0, 0, _log(rng, 16, 8192)])
    while B > 1 and B * (T + 1) > 64 * 8192:
        B = (B + 1) // 2
    # no more arithmetic than the largest listed case's
    while B > 1 and B * Tq * Hq * D * (P + T) > 32 * 64 * 32 * 128 * 10500:
        B = (B + 1) // 2
    if Tq * Hq * D * (P + T) > 32 * 64 * 32 * 128 * 10500:
        Tq = 1
    return {"op": op, "B": B, "Tq": Tq, "Hq": Hq, "Hkv": Hkv, "D": D, "P": P, "T": T, "dtype": dtype}


# ------------------------------------------------------------------ inputs


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dt)

    dt = DTYPES[case["dtype"]]
    B, Hkv, D, T = case["B"], case["Hkv"], case["D"], case["T"]
    s = {"op": case["op"], "k": normal(B, T, Hkv, D), "v": normal(B, T, Hkv, D)}
    if case["op"] == "evict":
        # accumulated weights: a few heavy keys, a long light tail, and keys that nothing has read yet
        u = torch.rand(B, Hkv, T, generator=g, device="cuda")
        z = torch.rand(B, Hkv, T, generator=g, device="cuda")
        s["scores"] = torch.where(z < 0.1, torch.zeros_like(u), (1e-4 + u) ** -0.7 - 0.99)
        low = max(1, T // 2) if case["ragged"] else T
        s.update(budget=case["budget"], window=case["window"], sink=case["sink"])
    else:
        Tq, Hq, P = case["Tq"], case["Hq"], case["P"]
        s["q"] = normal(B, Tq, Hq, D)
        s["kp"], s["vp"] = normal(P, Hkv, D), normal(P, Hkv, D)
        # the scores that some hundred earlier steps of this cache would have left
        if case["op"] == "scored":
            s["scores"] = torch.rand(B, Hkv, T, generator=g, device="cuda") * (100.0 * Hq / Hkv / T)
        low = max(Tq, T // 2)
    s["lengths"] = torch.randint(low, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    return s


def prepare(case, seed):
    if own:
        root = os.path.join(os.getcwd(), "latent-sparse-attention-rocm_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        import lsa_b200  # noqa: F401
    return _inputs(case, seed)


# ------------------------------------------------------------------ the operators


def _plain_attention(s):
    """(output, own keys' weights [B, Hkv, T]) in fp32."""
    q, k, v, kp, vp = (s[n].float() for n in ("q", "k", "v", "kp", "vp"))
    B, Tq, Hq, D = q.shape
    P, Hkv, _ = kp.shape
    T, G = k.shape[1], Hq // Hkv
    q = q.view(B, Tq, Hkv, G, D).permute(2, 0, 1, 3, 4) * D ** -0.5  # [Hkv, B, Tq, G, D]
    pre = (q.reshape(Hkv, B * Tq * G, D) @ kp.permute(1, 2, 0)).view(Hkv, B, Tq * G, P)
    mine = q.reshape(Hkv, B, Tq * G, D) @ k.permute(2, 0, 3, 1)  # [Hkv, B, Tq G, T]
    row = torch.arange(Tq, device=q.device).repeat_interleave(G)
    seen = s["lengths"].long()[:, None] - Tq + row[None, :] + 1  # own keys of each row [B, Tq G]
    hide = torch.arange(T, device=q.device)[None, None, :] >= seen[:, :, None]
    mine = mine.masked_fill(hide[None], -math.inf)
    both = torch.cat([pre, mine], dim=-1)
    top = both.amax(-1, keepdim=True)
    w = torch.exp(both - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total == 0, torch.ones_like(total), total)
    out = (w[..., :P].reshape(Hkv, B * Tq * G, P) @ vp.permute(1, 0, 2)).view(Hkv, B, Tq * G, D)
    out = out + w[..., P:] @ v.permute(2, 0, 1, 3)
    out = out.view(Hkv, B, Tq, G, D).permute(1, 2, 0, 3, 4).reshape(B, Tq, Hq, D)
    return out.to(s["q"].dtype), w[..., P:].sum(2).permute(1, 0, 2)


def _plain_evict(s):
    k, v, scores, n = s["k"], s["v"], s["scores"], s["lengths"].long()
    B, T, Hkv, D = k.shape
    C, window, sink = s["budget"], s["window"], s["sink"]
    j = torch.arange(T, device=k.device)[None, None, :]
    n_ = n[:, None, None]
    # the order of the scores as integers; the sinks and the window above every score
    bits = scores.contiguous().view(torch.int32).long()
    key = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF)
    key = torch.where((j < sink) | (j >= n_ - window), torch.full_like(key, 1 << 40), key)
    key = torch.where(j < n_, key, torch.full_like(key, -(1 << 40)))
    ids = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :C].sort(-1).values  # [B, Hkv, C]
    count = torch.minimum(n, torch.full_like(n, C))
    live = torch.arange(C, device=k.device)[None, None, :] < count[:, None, None]
    rows = ids.permute(0, 2, 1)[..., None].expand(B, C, Hkv, D)
    dead = ~live.permute(0, 2, 1)[..., None]
    kept = torch.gather(scores, 2, ids).masked_fill(~live, 0.0)
    return (torch.gather(k, 1, rows).masked_fill(dead, 0), torch.gather(v, 1, rows).masked_fill(dead, 0), kept,
            count.to(torch.int32), torch.where(live, ids, torch.full_like(ids, -1)).to(torch.int32))


def run(s):
    if own:
        import lsa_b200

        if s["op"] == "prefix":
            return lsa_b200.shared_prefix_attention(s["q"], s["kp"], s["vp"], s["k"], s["v"], s["lengths"])
        if s["op"] == "scored":
            return lsa_b200.scored_attention(s["q"], s["k"], s["v"], s["lengths"], s["scores"],
                                             k_prefix=s["kp"], v_prefix=s["vp"])
        e = lsa_b200.evict(s["k"], s["v"], s["scores"], s["lengths"], s["budget"], window_size=s["window"],
                           sink_size=s["sink"])
        return e.k, e.v, e.scores, e.lengths, e.ids
    if s["op"] == "prefix":
        return _plain_attention(s)[0]
    if s["op"] == "scored":
        out, weights = _plain_attention(s)
        T = s["scores"].shape[-1]
        live = torch.arange(T, device=out.device)[None, None, :] < s["lengths"].long()[:, None, None]
        return out, torch.where(live, s["scores"] + weights, s["scores"])
    return _plain_evict(s)


# ------------------------------------------------------------------ floors and 64 bits


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    B, Hkv, D, T = case["B"], case["Hkv"], case["D"], case["T"]
    if case["op"] == "evict":
        n = 0.75 * T if case["ragged"] else T
        kept = min(n, case["budget"])
        # the scores once; the kept rows in, the budget's rows, scores and ids out
        return {"bytes": B * Hkv * (4 * n + 2 * D * size * (kept + case["budget"]) + 8 * case["budget"]) + 8 * B,
                "flops": 0}
    Tq, Hq, P = case["Tq"], case["Hq"], case["P"]
    n = (max(Tq, T // 2) + T) / 2  # own keys of a sequence: between half a cache and all of it
    size_kv = 2 * Hkv * D * size
    nbytes = 2 * B * Tq * Hq * D * size + (P + B * n) * size_kv + 4 * B
    if case["op"] == "scored":
        nbytes += 8 * B * Hkv * T
    return {"bytes": nbytes, "flops": 4 * B * Tq * Hq * D * (P + n - (Tq - 1) / 2)}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "evict":
        return _exact_evict(s)
    B, Tq, Hq, D = s["q"].shape
    P, Hkv, _ = s["kp"].shape
    G = Hq // Hkv
    out = torch.zeros(B, Tq, Hq, D, dtype=torch.float64, device="cuda")
    scores = s["scores"].double() if case["op"] == "scored" else None
    for b in range(B):
        n = int(s["lengths"][b])
        key = torch.cat([s["kp"], s["k"][b, :n]]).double()
        val = torch.cat([s["vp"], s["v"][b, :n]]).double()
        last = P + n - Tq + torch.arange(Tq, device="cuda")
        allowed = torch.arange(P + n, device="cuda")[None, :] <= last[:, None]  # [Tq, P + n]
        for h in range(Hkv):
            q = s["q"][b, :, h * G:(h + 1) * G].double()  # [Tq, G, D]
            logits = (q.reshape(Tq * G, D) @ key[:, h].T).view(Tq, G, P + n) / math.sqrt(D)
            p = torch.softmax(logits.masked_fill(~allowed[:, None, :], -math.inf), dim=-1)
            p = torch.nan_to_num(p)  # a row that sees no key
            out[b, :, h * G:(h + 1) * G] = (p.view(Tq * G, P + n) @ val[:, h]).view(Tq, G, D)
            if scores is not None:
                scores[b, h, :n] += p[..., P:].sum((0, 1))
    return out if scores is None else (out, scores)


def _exact_evict(s):
    """Each row's ids by counting how many candidates go before each of them."""
    k, v, scores = s["k"], s["v"], s["scores"].double()
    B, T, Hkv, D = k.shape
    C, window, sink = s["budget"], s["window"], s["sink"]
    ko = torch.zeros(B, C, Hkv, D, dtype=torch.float64, device="cuda")
    vo, so = torch.zeros_like(ko), torch.zeros(B, Hkv, C, dtype=torch.float64, device="cuda")
    ids = torch.full((B, Hkv, C), -1, dtype=torch.int32, device="cuda")
    counts = []
    for b in range(B):
        n = int(s["lengths"][b])
        counts.append(min(n, C))
        for h in range(Hkv):
            keep = torch.ones(n, dtype=torch.bool, device="cuda")
            if n > C:
                mid, need = scores[b, h, sink:n - window], C - sink - window
                keep[sink:n - window] = False
                if need:
                    cut = torch.kthvalue(mid, mid.numel() - need + 1).values  # the last score that stays
                    above = mid > cut
                    level = (mid == cut).nonzero()[:need - int(above.sum()), 0]
                    keep[sink + above.nonzero()[:, 0]] = True
                    keep[sink + level] = True
            at = keep.nonzero()[:, 0]
            ids[b, h, :at.numel()] = at.int()
            ko[b, :at.numel(), h], vo[b, :at.numel(), h] = k[b, at, h].double(), v[b, at, h].double()
            so[b, h, :at.numel()] = scores[b, h, at]
    return ko, vo, so, torch.tensor(counts, dtype=torch.int32, device="cuda"), ids
