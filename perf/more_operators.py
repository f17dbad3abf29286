"""Cases of a paged cache held in 8 bits: what fills it, what reads it, what moves its pages.

Five operators of a serving loop: the norms and the rotation of a step's queries and keys; the
append of keys and values to pages of 8-bit codes with one scale a (page, KV head); attention
over the pages; the same over a selected list of positions; copies of whole pages.

``own`` false: the plain forms, elementary torch operations in fp32 (angles in fp64). ``own``
true: the calls a user makes of ``lsa_b200``.

A cache is k, v [pages, Hkv, page, D] codes (e4m3 or int8) and k_scale, v_scale [pages, Hkv] fp32;
page_table [B, M] int32 maps a sequence's tokens to its pages, -1 past them; lengths [B] count
the tokens of a sequence, those of the call among them.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
EPS = 1e-6


# ------------------------------------------------------------------ cases


def listed():
    heads = {"Hq": 32, "Hkv": 8, "D": 128}
    return [
        # --- norms and rotation
        # a decode batch: 64 tokens, where the launch counts
        {"name": "rotate_decode_64", "op": "rotate", "B": 64, "T": 1, **heads, "R": 128, "interleaved": False,
         "norm": True, "scaling": "none", "dtype": "bf16", "far": 32768},
        # two prompts of a long-context model, frequencies blended for 8 times the trained length
        {"name": "rotate_prompt_2x16k", "op": "rotate", "B": 2, "T": 16384, **heads, "R": 128, "interleaved": False,
         "norm": True, "scaling": "yarn", "dtype": "bf16", "far": 131072},
        # --- append
        # one token a sequence, into pages that are partly full
        {"name": "append_decode_64", "op": "append", "B": 64, "Tq": 1, **heads, "T": 1024, "page": 64,
         "code": "e4m3", "ragged": True, "idle": False, "dtype": "bf16"},
        # four ragged prompts
        {"name": "append_prompt_4x16k", "op": "append", "B": 4, "Tq": 16383, **heads, "T": 16384, "page": 64,
         "code": "e4m3", "ragged": True, "idle": False, "dtype": "bf16"},
        # --- attention
        # a few short requests: the latency of one decode step
        {"name": "attend_decode_4x2k", "op": "attend", "B": 4, "Tq": 1, **heads, "T": 2048, "page": 64,
         "code": "e4m3", "ragged": True, "idle": False, "dtype": "bf16"},
        # a full decode batch
        {"name": "attend_decode_64x8k", "op": "attend", "B": 64, "Tq": 1, **heads, "T": 8191, "page": 64,
         "code": "e4m3", "ragged": True, "idle": False, "dtype": "bf16"},
        # one very long sequence, 8-bit integers
        {"name": "attend_decode_1x128k", "op": "attend", "B": 1, "Tq": 1, **heads, "T": 131072, "page": 128,
         "code": "int8", "ragged": False, "idle": False, "dtype": "fp16"},
        # chunks of two long prompts against what is cached: the compute-bound end
        {"name": "attend_chunk_2x1024", "op": "attend", "B": 2, "Tq": 1024, **heads, "T": 16384, "page": 64,
         "code": "e4m3", "ragged": True, "idle": False, "dtype": "bf16"},
        # --- the read of selected positions
        # one sequence's decode step: 2048 selected keys, the window and the sinks
        {"name": "read_decode_1x32k", "op": "read", "B": 1, **heads, "T": 32768, "page": 64, "W": 2116,
         "code": "e4m3", "ragged": False, "idle": False, "dtype": "bf16"},
        # a batch of them
        {"name": "read_decode_32x32k", "op": "read", "B": 32, **heads, "T": 32768, "page": 64, "W": 2116,
         "code": "e4m3", "ragged": True, "idle": False, "dtype": "bf16"},
        # --- pages
        # 16 sequences forked: the copies of their last, partly full pages
        {"name": "move_fork_16", "op": "move", "n": 16, "pages": 1024, "Hkv": 8, "D": 128, "page": 64, "code": "e4m3"},
        # a pool compacted
        {"name": "move_compact_4k", "op": "move", "n": 4000, "pages": 8192, "Hkv": 8, "D": 128, "page": 64,
         "code": "e4m3"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotate", "append", "attend", "attend", "attend", "read", "move"])
    Hkv, D = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128])
    Hq = Hkv * rng.choice([1, 2, 3, 4, 4, 6, 8, 8])
    dtype, code = rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["e4m3", "e4m3", "int8"])
    page = rng.choice([16, 32, 64, 64, 128])
    if op == "rotate":
        B, T = rng.choice([(_log(rng, 1, 256), 1), (_log(rng, 1, 8), _log(rng, 2, 16384))])
        D = rng.choice([64, 128, 128, 256])
        while B > 1 and B * T * (Hq + Hkv) * D > 2 * 16384 * 40 * 128:
            B = (B + 1) // 2
        while B * T * (Hq + Hkv) * D > 2 * 16384 * 40 * 128:
            T = (T + 1) // 2
        return {"op": op, "B": B, "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "R": rng.choice([D, D, D // 2, D // 4]),
                "interleaved": rng.random() < 0.4, "norm": rng.random() < 0.7,
                "scaling": rng.choice(["none", "none", "linear", "yarn"]),
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "far": rng.choice([4096, 32768, 131072, 1048576])}
    if op == "move":
        pages = _log(rng, 64, 16384)
        while pages * Hkv * D * page > 8192 * 8 * 128 * 64:
            pages //= 2
        return {"op": op, "n": _log(rng, 1, pages // 2), "pages": pages, "Hkv": Hkv, "D": D, "page": page,
                "code": code}
    ragged, idle = rng.random() < 0.7, rng.random() < 0.3
    B = _log(rng, 1, 64)
    case = {"op": op, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "code": code, "ragged": ragged, "idle": idle,
            "dtype": dtype}
    if op == "append":
        Tq = rng.choice([1, 1, 2, 5, _log(rng, 8, 16383), _log(rng, 8, 16383)])
        T = Tq + _log(rng, 1, 1024)
        while B > 1 and B * T > 4 * 16384:
            B = (B + 1) // 2
        return {**case, "B": B, "Tq": Tq, "T": T}
    T = _log(rng, 64, 131072)
    while B > 1 and B * T > 32 * 32768:
        B = (B + 1) // 2
    if op == "read":
        W = min(T, _log(rng, 68, 4096))
        while B > 1 and B * W > 32 * 2116:
            B = (B + 1) // 2
        return {**case, "B": B, "T": T, "W": W}
    Tq = min(T, rng.choice([1, 1, 1, 2, 3, 5, 8, 32, 61, _log(rng, 64, 1024)]))
    # no more than the largest listed case's bytes and arithmetic
    while B > 1 and (B * (T + 1) > 64 * 8192 or B * Tq * Hq * T > 2 * 1024 * 32 * 16384):
        B = (B + 1) // 2
    while Tq * Hq * T > 2 * 1024 * 32 * 16384:
        Tq = (Tq + 1) // 2
    return {**case, "B": B, "Tq": Tq, "T": T}


# ------------------------------------------------------------------ inputs


def _power_scale(top, code):
    """The smallest power of two s >= 2^-60 with top <= (the code's largest value) * s."""
    fraction, e = torch.frexp(top)  # top = fraction * 2^e, fraction in [0.5, 1)
    if code == "e4m3":  # 448 = 0.875 * 2^9
        e = torch.where(fraction <= 0.875, e - 9, e - 8)
    else:  # 127 = 0.9921875 * 2^7
        e = torch.where(fraction <= 0.9921875, e - 7, e - 6)
    e = torch.where(top > 0, e, torch.full_like(e, -60)).clamp(min=-60)
    return ((e.int() + 127) << 23).view(torch.float32)


def _encode(x, code):
    """fp32 values in units of their scale -> codes, to the nearest (ties to even)."""
    if code == "e4m3":
        return x.to(torch.float8_e4m3fn)
    return x.round().clamp(-127, 127).to(torch.int8)


def _pool(g, pages, Hkv, page, D, code, gain):
    """Codes and scales of pages of normal values, each channel of a head with a gain of its own."""
    codes = torch.empty(pages, Hkv, page, D, dtype=CODES[code], device="cuda")
    scale = torch.empty(pages, Hkv, dtype=torch.float32, device="cuda")
    step = max(1, (1 << 27) // (Hkv * page * D))
    for a in range(0, pages, step):
        b = min(pages, a + step)
        x = torch.randn(b - a, Hkv, page, D, generator=g, device="cuda").mul_(gain)
        s = _power_scale(x.abs().amax((2, 3)), code)
        scale[a:b] = s
        codes[a:b] = _encode(x.div_(s[..., None, None]), code)
    return codes, scale


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op = case["op"]
    s = {"op": op}
    if op == "rotate":
        dt, B, T, D, R = DTYPES[case["dtype"]], case["B"], case["T"], case["D"], case["R"]
        # q and k as a projection leaves them: slices of one row a token
        qkv = torch.randn(B, T, case["Hq"] + 2 * case["Hkv"], D, generator=g, device="cuda").to(dt)
        s["q"], s["k"] = qkv[:, :, :case["Hq"]], qkv[:, :, case["Hq"]:case["Hq"] + case["Hkv"]]
        first = torch.randint(0, max(1, case["far"] - T), (B, 1), generator=g, device="cuda")
        s["positions"] = (first + torch.arange(T, device="cuda")).to(torch.int32)
        s["frequencies"], s["amplitude"] = _frequencies(R, case["scaling"])
        s["interleaved"], s["norm"] = case["interleaved"], case["norm"]
        s["qw"] = (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(dt)
        s["kw"] = (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(dt)
        return s
    Hkv, D, page, code = case["Hkv"], case["D"], case["page"], case["code"]
    s["code"] = code
    gain = torch.exp(0.5 * torch.randn(Hkv, 1, D, generator=g, device="cuda"))
    if op == "move":
        P = case["pages"]
    else:
        B, M = case["B"], -(-case["T"] // page)
        P = B * M + 1  # page 0 is no one's
    s["k8"], s["ks"] = _pool(g, P, Hkv, page, D, code, gain)
    s["v8"], s["vs"] = _pool(g, P, Hkv, page, D, code, 1.0)
    if op == "move":
        ids = torch.randperm(P, generator=g, device="cuda")[:2 * case["n"]].to(torch.int32)
        s["src"], s["dst"] = ids[:case["n"]].contiguous(), ids[case["n"]:].contiguous()
        return s
    dt, T, Tq = DTYPES[case["dtype"]], case["T"], case.get("Tq", 1)
    low = max(Tq, T // 2) if case["ragged"] else T
    lengths = torch.randint(low, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    if case["idle"]:  # a place of the batch that no request holds
        lengths[0] = 0
    s["lengths"] = lengths
    table = 1 + torch.randperm(B * M, generator=g, device="cuda").view(B, M)  # an allocator's state after churn
    unused = torch.arange(M, device="cuda") * page >= lengths[:, None]
    s["table"] = table.masked_fill(unused, -1).to(torch.int32)
    if op == "append":
        s["k"] = (torch.randn(B, Tq, Hkv, D, generator=g, device="cuda") * gain.view(Hkv, D)).to(dt)
        s["v"] = torch.randn(B, Tq, Hkv, D, generator=g, device="cuda").to(dt)
        return s
    s["q"] = torch.randn(B, Tq, case["Hq"], D, generator=g, device="cuda").to(dt)
    if op == "read":
        # the sinks, the window and positions spread over the rest, in no order: what a selection lists
        W, n = case["W"], lengths.double()[:, None]
        far = W - min(W // 2, 64)
        j = torch.arange(W, device="cuda", dtype=torch.float64)
        spread = (j + torch.rand(B, W, generator=g, device="cuda", dtype=torch.float64)) * (n - (W - far)) / far
        ids = torch.where(j < far, spread.floor(), n - W + j)
        ids = torch.where(n > W, ids, j.expand(B, W))
        s["lists"] = ids[:, torch.randperm(W, generator=g, device="cuda")].to(torch.int32).contiguous()
        few = (lengths <= W)[:, None]
        s["lists"] = torch.where(few, j.expand(B, W).to(torch.int32), s["lists"])
        s["counts"] = lengths.clamp(max=W)
        s["rows"] = torch.arange(B, device="cuda", dtype=torch.int32)
    return s


def _frequencies(R, scaling, base=10000.0, factor=8.0, trained=16384):
    """(inverse frequencies, radians a position, fp64 [R / 2], amplitude)."""
    i = torch.arange(R // 2, device="cuda", dtype=torch.float64)
    f = base ** (-2.0 * i / R)
    if scaling == "none":
        return f, 1.0
    if scaling == "linear":
        return f / factor, 1.0
    # blended: dimensions that turn often within the trained length keep their frequency
    def dim(turns):
        return R * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(math.floor(dim(32.0)), 0), min(math.ceil(dim(1.0)), R - 1)
    ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0


def prepare(case, seed):
    return _inputs(case, seed)


# ------------------------------------------------------------------ the operators


def _plain_rotate(s):
    R = 2 * s["frequencies"].numel()
    angle = s["positions"].double()[..., None] * s["frequencies"]  # [B, T, R / 2]
    cos = (angle.cos() * s["amplitude"]).float()[:, :, None, :]
    sin = (angle.sin() * s["amplitude"]).float()[:, :, None, :]

    def one(x, weight):
        y = x.float()
        if s["norm"]:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()
        if s["interleaved"]:
            a, b = y[..., 0:R:2], y[..., 1:R:2]
            turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        else:
            a, b = y[..., :R // 2], y[..., R // 2:R]
            turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        return torch.cat([turned, y[..., R:]], -1).to(x.dtype)

    return one(s["q"], s["qw"]), one(s["k"], s["kw"])


def _plain_append(s):
    lengths, table, code = s["lengths"].long(), s["table"].long(), s["code"]
    B, Tq, Hkv, D = s["k"].shape
    page, M = s["k8"].shape[2], table.shape[1]
    first = (lengths - Tq).clamp(min=0)  # the new tokens are [first, lengths)
    J = min(M, (Tq + page - 2) // page + 1)  # pages that Tq tokens touch at most
    slot = (first // page)[:, None] + torch.arange(J, device=table.device)  # [B, J]
    touched = (slot < M) & (slot * page < lengths[:, None])
    at = torch.gather(table, 1, slot.clamp(max=M - 1))
    at = torch.where(touched, at, torch.zeros_like(at))  # page 0: no one's
    t = slot[..., None] * page + torch.arange(page, device=table.device)  # [B, J, page]
    new = touched[..., None] & (t >= first[:, None, None]) & (t < lengths[:, None, None])
    old = touched[..., None] & (t < first[:, None, None])
    token = (t - (lengths - Tq)[:, None, None]).clamp(0, Tq - 1)
    batch = torch.arange(B, device=table.device)[:, None, None]
    new_, old_ = new[:, :, None, :, None], old[:, :, None, :, None]

    def one(x, codes, scale):
        x = x[batch, token].permute(0, 1, 3, 2, 4).float()  # [B, J, Hkv, page, D]
        was = scale[at]
        needed = _power_scale(x.abs().masked_fill(~new_, 0.0).amax((3, 4)), code)
        now = torch.where(old.any(-1)[..., None], torch.maximum(was, needed), needed)
        now = torch.where(new.any(-1)[..., None], now, was)
        before = codes[at]
        again = _encode(before.float() * was[..., None, None] / now[..., None, None], code)
        fresh = _encode(x / now[..., None, None], code)
        byte = before.view(torch.int8)
        byte = torch.where(old_, again.view(torch.int8), byte)
        byte = torch.where(new_, fresh.view(torch.int8), byte)
        codes.view(torch.int8)[at] = byte
        scale[at] = now

    one(s["k"], s["k8"], s["ks"])
    one(s["v"], s["v8"], s["vs"])
    return s["k8"], s["v8"], s["ks"], s["vs"]


def _plain_softmax(x):
    top = x.amax(-1, keepdim=True)
    w = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = w.sum(-1, keepdim=True)
    return w / torch.where(total == 0, torch.ones_like(total), total)


def _plain_attend(s):
    q, lengths = s["q"], s["lengths"].long()
    B, Tq, Hq, D = q.shape
    Hkv, page = s["k8"].shape[1:3]
    G, M = Hq // Hkv, s["table"].shape[1]
    at = s["table"].long().clamp(min=0)

    def whole(codes, scale):  # [B, Hkv, M page, D]
        x = codes[at].float().mul_(scale[at][..., None, None])
        return x.permute(0, 2, 1, 3, 4).reshape(B, Hkv, M * page, D)

    rows = (q.float() * D ** -0.5).view(B, Tq, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, Tq * G, D)
    logits = rows @ whole(s["k8"], s["ks"]).transpose(-1, -2)
    row = torch.arange(Tq, device=q.device).repeat_interleave(G)
    seen = lengths[:, None] - Tq + row + 1  # keys of each row [B, Tq G]
    hide = torch.arange(M * page, device=q.device) >= seen[..., None]
    w = _plain_softmax(logits.masked_fill_(hide[:, None], -math.inf))
    values = whole(s["v8"], s["vs"]).masked_fill_(
        (torch.arange(M * page, device=q.device) >= lengths[:, None])[:, None, :, None], 0.0)
    out = (w @ values).view(B, Hkv, Tq, G, D).permute(0, 2, 1, 3, 4)
    return out.reshape(B, Tq, Hq, D).to(q.dtype)


def _plain_read(s):
    q, ids, lengths = s["q"], s["lists"].long(), s["lengths"].long()
    R, _, Hq, D = q.shape
    Hkv, page = s["k8"].shape[1:3]
    W = ids.shape[1]
    row = s["rows"].long()
    live = (torch.arange(W, device=q.device) < s["counts"][:, None]) & (ids < lengths[row][:, None])
    ids = torch.where(live, ids, torch.zeros_like(ids))
    at = torch.gather(s["table"].long()[row], 1, ids // page).clamp(min=0)

    def listed_rows(codes, scale):  # [R, Hkv, W, D]
        return codes[at, :, ids % page].float().mul_(scale[at][..., None]).permute(0, 2, 1, 3)

    rows = (q.float() * D ** -0.5).view(R, Hkv, Hq // Hkv, D)
    logits = rows @ listed_rows(s["k8"], s["ks"]).transpose(-1, -2)
    w = _plain_softmax(logits.masked_fill_(~live[:, None, None], -math.inf))
    values = listed_rows(s["v8"], s["vs"]).masked_fill_(~live[:, None, :, None], 0.0)
    return (w @ values).reshape(R, 1, Hq, D).to(q.dtype)


def _plain_move(s):
    src, dst = s["src"].long(), s["dst"].long()
    for name in ("k8", "v8"):
        codes = s[name].view(torch.int8)
        codes[dst] = codes[src]
    for name in ("ks", "vs"):
        s[name][dst] = s[name][src]
    return s["k8"], s["v8"], s["ks"], s["vs"]


def run(s):
    op = s["op"]
    if own:
        if "lsa_b200" not in sys.modules:
            sys.path.insert(0, os.path.join(os.getcwd(), "latent-sparse-attention-rocm_b200"))
        import lsa_b200

        if op == "rotate":
            return lsa_b200.norm_rotate(s["q"], s["k"], s["positions"], s["frequencies"],
                                        s["qw"] if s["norm"] else None, s["kw"] if s["norm"] else None, eps=EPS,
                                        interleaved=s["interleaved"], amplitude=s["amplitude"])
        pages = lsa_b200.QuantizedPages(s["k8"], s["v8"], s["ks"], s["vs"])
        if op == "append":
            lsa_b200.append_quantized(pages, s["k"], s["v"], s["table"], s["lengths"])
        elif op == "move":
            lsa_b200.move_pages(pages, s["src"], s["dst"])
        elif op == "attend":
            return lsa_b200.quantized_attention(s["q"], pages, s["table"], s["lengths"])
        else:
            return lsa_b200.quantized_read(s["q"], pages, s["table"], s["lengths"], s["lists"], s["counts"],
                                           s["rows"])
        return s["k8"], s["v8"], s["ks"], s["vs"]
    plain = {"rotate": _plain_rotate, "append": _plain_append, "attend": _plain_attend, "read": _plain_read,
             "move": _plain_move}
    return plain[op](s)


# ------------------------------------------------------------------ floors and 64 bits


def work(case):
    op, Hkv, D = case["op"], case["Hkv"], case["D"]
    if op == "rotate":
        size = 4 if case["dtype"] == "fp32" else 2
        n = case["B"] * case["T"]
        values = n * (case["Hq"] + Hkv) * D
        return {"bytes": 2 * size * values + 4 * n + 4 * case["R"] + (2 * size * D if case["norm"] else 0),
                "flops": (10 if case["norm"] else 6) * values}
    page = case["page"]
    if op == "move":
        return {"bytes": 4 * case["n"] * Hkv * (page * D + 4) + 8 * case["n"], "flops": 0}
    B, T, Tq = case["B"], case["T"], case.get("Tq", 1)
    busy = B - 1 if case["idle"] else B
    low = max(Tq, T // 2) if case["ragged"] else T
    n = (low + T) / 2  # tokens of a sequence
    if op == "append":
        rows = busy * Tq * Hkv
        pages = busy * Hkv * (1 if Tq == 1 else (Tq + page - 1) / page + 1)
        return {"bytes": 2 * rows * D * 3 + 2 * 8 * pages + 4 * B + 4 * pages / Hkv, "flops": 6 * rows * D}
    if op == "read":
        n, Tq = min(case["W"], n), 1
        nbytes = busy * n * (2 * Hkv * D + 4)  # the rows' codes and the list
        scales = min(n, T / page) * busy * Hkv * 8
    else:
        nbytes = busy * n * 2 * Hkv * D
        scales = busy * (n / page) * (Hkv * 8 + 4)
    return {"bytes": nbytes + scales + 4 * B * Tq * case["Hq"] * D + 4 * B,
            "flops": 4 * busy * Tq * case["Hq"] * D * max(n - (Tq - 1) / 2, 1)}


def exact(case, seed):
    if case["op"] == "move":
        return None
    s = _inputs(case, seed)
    return {"rotate": _exact_rotate, "append": _exact_append, "attend": _exact_attend,
            "read": _exact_read}[case["op"]](s)


def _exact_rotate(s):
    """Pairs as complex numbers, turned by a product with e^(i angle)."""
    R = 2 * s["frequencies"].numel()
    turn = torch.polar(torch.full((), s["amplitude"], dtype=torch.float64, device="cuda"),
                       s["positions"].double().unsqueeze(-1) * s["frequencies"])[:, :, None]
    got = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        y = x.double()
        if s["norm"]:
            y = y / torch.sqrt(torch.square(y).sum(-1, keepdim=True) / y.shape[-1] + EPS) * w.double()
        head = y[..., :R]
        pairs = head.unflatten(-1, (R // 2, 2)) if s["interleaved"] else head.unflatten(-1, (2, R // 2)).transpose(-1, -2)
        turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        if not s["interleaved"]:
            turned = turned.transpose(-1, -2)
        y[..., :R] = turned.flatten(-2)
        got.append(y)
    return tuple(got)


def _grid(code):
    """The values that a code can have, ascending, and whether the code's last bit is 0."""
    if code == "int8":
        v = torch.arange(-127, 128, dtype=torch.float64, device="cuda")
        return v, v % 2 == 0
    mags = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)]
    mags = mags[:-1]  # the last code is NaN
    v = torch.tensor([-m for m in reversed(mags[1:])] + mags, dtype=torch.float64, device="cuda")
    even = [i % 2 == 0 for i in range(len(mags))]
    return v, torch.tensor(list(reversed(even[1:])) + even, device="cuda")


def _nearest(x, code):
    v, even = _grid(code)
    hi = torch.searchsorted(v, x.contiguous()).clamp(1, v.numel() - 1)
    below, above = x - v[hi - 1], v[hi] - x
    up = (above < below) | ((above == below) & even[hi])
    return v[torch.where(up, hi, hi - 1)]


def _exact_append(s):
    """Page by page of each sequence, every scale searched from the smallest power of two up."""
    code, table = s["code"], s["table"].tolist()
    qmax = 448.0 if code == "e4m3" else 127.0
    B, Tq, Hkv, D = s["k"].shape
    page = s["k8"].shape[2]
    powers = torch.tensor([2.0 ** e for e in range(-60, 121)], dtype=torch.float64, device="cuda")
    got = []
    for x, codes, scale in ((s["k"], s["k8"], s["ks"]), (s["v"], s["v8"], s["vs"])):
        codes, scale = codes.double(), scale.double()
        for b, n in enumerate(s["lengths"].tolist()):
            first = max(0, n - Tq)
            for j in range(first // page, -(-n // page) if n else 0):
                p, a, z = table[b][j], max(first, j * page), min(n, (j + 1) * page)
                rows = x[b, a - (n - Tq):z - (n - Tq)].double().transpose(0, 1)  # [Hkv, tokens, D]
                now = powers[torch.searchsorted(powers * qmax, rows.abs().amax((1, 2)).contiguous())]
                kept = a - j * page
                if kept:
                    was = scale[p]
                    now = torch.maximum(now, was)
                    codes[p, :, :kept] = _nearest(codes[p, :, :kept] * (was / now)[:, None, None], code)
                codes[p, :, kept:z - j * page] = _nearest(rows / now[:, None, None], code)
                scale[p] = now
        got.append((codes, scale))
    return got[0][0], got[1][0], got[0][1], got[1][1]


def _keys(s, b, ids):
    """Keys and values [n, Hkv, D] of table row b at the positions ids, in 64 bits."""
    page = s["k8"].shape[2]
    p, o = s["table"][b].long()[ids // page], ids % page
    return (s["k8"][p, :, o].double() * s["ks"][p].double()[..., None],
            s["v8"][p, :, o].double() * s["vs"][p].double()[..., None])


def _exact_attend(s):
    B, Tq, Hq, D = s["q"].shape
    G = Hq // s["k8"].shape[1]
    out = torch.zeros(B, Tq, Hq, D, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lengths"].tolist()):
        if n == 0:
            continue
        key, val = _keys(s, b, torch.arange(n, device="cuda"))
        allowed = torch.arange(n, device="cuda") <= (n - Tq + torch.arange(Tq, device="cuda"))[:, None]
        for h in range(Hq):
            logits = s["q"][b, :, h].double() @ key[:, h // G].T / math.sqrt(D)
            p = torch.softmax(logits.masked_fill(~allowed, -math.inf), -1)
            out[b, :, h] = torch.nan_to_num(p) @ val[:, h // G]  # a row without a key: zeros
    return out


def _exact_read(s):
    R, _, Hq, D = s["q"].shape
    G = Hq // s["k8"].shape[1]
    out = torch.zeros(R, 1, Hq, D, dtype=torch.float64, device="cuda")
    for r, b in enumerate(s["rows"].tolist()):
        ids = s["lists"][r, :int(s["counts"][r])].long()
        if ids.numel() == 0:
            continue
        key, val = _keys(s, b, ids)
        for h in range(Hq):
            p = torch.softmax(key[:, h // G] @ s["q"][r, 0, h].double() / math.sqrt(D), 0)
            out[r, 0, h] = p @ val[:, h // G]
    return out
