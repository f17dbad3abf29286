"""The 8-bit paged cache's operators from their definitions, in 64 bits on the CPU, and pools to test them on."""

import math

import torch

CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
QMAX = {"e4m3": 448.0, "int8": 127.0}


def code_name(pages):
    return "int8" if pages.k.dtype == torch.int8 else "e4m3"


def grid(code):
    """Every value that a code has, ascending, and its code's last bit."""
    if code == "int8":
        v = torch.arange(-127, 128, dtype=torch.float64)
        return v, v.long() & 1
    bits = torch.arange(0, 127, dtype=torch.uint8)
    mags = bits.view(torch.float8_e4m3fn).double()
    v = torch.cat([-mags[1:].flip(0), mags])
    last = torch.cat([bits[1:].flip(0), bits]).long() & 1
    return v, last


def nearest(x, code):
    """x (64 bits) to the nearest code's value, ties to the code whose last bit is 0."""
    v, last = grid(code)
    hi = torch.searchsorted(v, x.contiguous()).clamp(1, v.numel() - 1)
    below, above = x - v[hi - 1], v[hi] - x
    up = (above < below) | ((above == below) & (last[hi] == 0))
    return v[torch.where(up, hi, hi - 1)]


def scale_for(top, code):
    e = -60
    while top > QMAX[code] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def append(pages, k, v, table, lengths, counts=None):
    """append_quantized on CPU tensors, one token at a time of each (sequence, page, head)."""
    code = code_name(pages)
    B, Tq, Hkv, D = k.shape
    P, page, M = pages.k.shape[0], pages.k.shape[2], table.shape[1]
    for x, codes, scale in ((k, pages.k, pages.k_scale), (v, pages.v, pages.v_scale)):
        for b in range(B):
            n = int(lengths[b])
            first = max(0, n - (Tq if counts is None else min(Tq, max(0, int(counts[b])))))
            for slot in range(first // page, min(M, -(-max(n, 0) // page))):
                p, a, z = int(table[b, slot]), max(first, slot * page), min(n, slot * page + page)
                if not 0 <= p < P or z <= a:
                    continue
                for h in range(Hkv):
                    new = x[b, a - (n - Tq):z - (n - Tq), h].double()
                    now, kept = scale_for(float(new.abs().max()), code), a - slot * page
                    if kept:
                        was = float(scale[p, h])
                        now = max(was, now)
                        old = codes[p, h, :kept].double() * (was / now)
                        codes[p, h, :kept] = nearest(old, code).to(codes.dtype)
                    codes[p, h, kept:z - slot * page] = nearest(new / now, code).to(codes.dtype)
                    scale[p, h] = now


def move(pages, src, dst):
    P = pages.k.shape[0]
    for s, d in zip(src.tolist(), dst.tolist()):
        if 0 <= s < P and 0 <= d < P:
            for t in pages:
                t = t.view(torch.int8) if t.element_size() == 1 else t
                t[d] = t[s]


def keys(pages, table_row, ids):
    """(ids on mapped pages, their keys and values [n, Hkv, D] in 64 bits)."""
    P, page = pages.k.shape[0], pages.k.shape[2]
    ids = ids[(ids >= 0) & (ids < table_row.numel() * page)]
    p = table_row.long()[ids // page]
    ids = ids[(p >= 0) & (p < P)]
    p, o = table_row.long()[ids // page], ids % page
    return (ids, pages.k[p, :, o].double() * pages.k_scale[p].double()[..., None],
            pages.v[p, :, o].double() * pages.v_scale[p].double()[..., None])


def rows(q, key, val, scale, seen, half):
    """Rows q [n, D] of one head: (output, lse, how far off a kernel may be). `seen` [n, keys].

    Off: the weights are rounded to 16 bits (`half` of each), the logits are fp32 sums of D products of exact
    factors (at most D + 4 roundings of 2^-24 of the sum of magnitudes, and what q loses where it is made fp16:
    2^-33 of its largest value a product), an error d of a logit changes a weight and the sum by 2^d - 1 each; exponentials,
    sums and joins: 2^-20; the output is rounded once."""
    logits = q @ key.T * scale
    logits = logits.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(logits, -1) if key.shape[0] else torch.full((q.shape[0],), -math.inf, dtype=torch.float64)
    w = torch.exp(logits - torch.where(lse == -math.inf, 0.0, lse)[:, None])
    out = w @ val
    if not key.shape[0]:
        return out, lse, torch.zeros_like(out), torch.zeros_like(lse)
    D = q.shape[1]
    size = (q.abs() @ key.abs().T * scale).masked_fill(~seen, 0.0).amax(-1)
    lost = D * 2.0 ** -33 * q.abs().amax(-1) * key.abs().max() * scale
    d = (D + 4) * 2.0 ** -24 * size + lost  # of a natural logit
    off = (w @ val.abs()) * (half + 2 * d + 2.0 ** -20)[:, None] + half * out.abs()
    off = off + 2.0 ** -36 * val.abs().max() + 2.0 ** -24  # weights, and fp16 outputs, below the smallest normal
    return out, lse, off, d + 2.0 ** -20 + 2.0 ** -22 * lse.abs().nan_to_num(posinf=0.0)


def attention(q, pages, table, lengths, scale=None):
    """(out, lse, off, lse_off), all 64 bits."""
    B, Tq, Hq, D = q.shape
    G = Hq // pages.k.shape[1]
    half = torch.finfo(q.dtype).eps / 2
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, Tq, Hq, D, dtype=torch.float64)
    off = torch.zeros_like(out)
    lse = torch.zeros(B, Tq, Hq, dtype=torch.float64)
    lse_off = torch.zeros_like(lse)
    for b in range(B):
        n = max(int(lengths[b]), 0)
        ids, key, val = keys(pages, table[b], torch.arange(n))
        seen = ids[None, :] < (n - Tq + torch.arange(Tq) + 1)[:, None]
        for h in range(Hq):
            r = rows(q[b, :, h].double(), key[:, h // G], val[:, h // G], scale, seen, half)
            out[b, :, h], lse[b, :, h], off[b, :, h], lse_off[b, :, h] = r
    return out, lse, off, lse_off


def read(q, pages, table, lengths, lists, counts, table_rows, scale=None):
    R, _, Hq, D = q.shape
    G = Hq // pages.k.shape[1]
    half = torch.finfo(q.dtype).eps / 2
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(R, 1, Hq, D, dtype=torch.float64)
    off = torch.zeros_like(out)
    for r in range(R):
        row = int(table_rows[r])
        if not 0 <= row < table.shape[0]:
            continue
        ids = lists[r, :max(0, min(int(counts[r]), lists.shape[1]))].long()
        ids = ids[(ids >= 0) & (ids < int(lengths[row]))]
        ids, key, val = keys(pages, table[row], ids)
        seen = torch.ones(1, ids.numel(), dtype=torch.bool)
        for h in range(Hq):
            out[r, :, h], _, off[r, :, h], _ = rows(q[r, :, h].double(), key[:, h // G], val[:, h // G], scale, seen, half)
    return out, off


def pool(g, n, Hkv, page, D, code, spread=2.0):
    """A pool of normal values on the CPU, every (page, head) at a size of its own."""
    from lsa_b200 import QuantizedPages

    pages = QuantizedPages.new(n, Hkv, page, D, CODES[code], "cpu")
    for codes, scale in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)):
        x = torch.randn(n, Hkv, page, D, generator=g)
        s = x.abs().amax((2, 3)) / QMAX[code]
        codes.copy_(nearest(x.double() / s[..., None, None].double(), code).to(codes.dtype))
        # scales of the size that makes the values about 1, and not powers of two
        scale.copy_(s * torch.exp2((torch.rand(n, Hkv, generator=g) - 0.5) * spread))
    return pages


def paged(g, lengths, page, spare=3):
    """A page table [B, M] of shuffled pages for the lengths, -1 past them, and the pool's page count."""
    M = max([-(-n // page) for n in lengths] + [1])
    held = [-(-n // page) for n in lengths]
    total = sum(held) + spare
    order = torch.randperm(total, generator=g)
    table = torch.full((len(lengths), M), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    return table, total


def poison(pages, table, lengths):
    """What lies behind the sequences' last tokens, and on pages that no one holds, becomes NaN (e4m3) or the largest code."""
    bad = 0x7F
    P, page = pages.k.shape[0], pages.k.shape[2]
    mine = torch.zeros(P, page, dtype=torch.bool)
    for b, n in enumerate(lengths):
        for slot in range(-(-n // page)):
            p = int(table[b, slot])
            if 0 <= p < P:
                mine[p, :min(page, n - slot * page)] = True
    for codes, scale in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)):
        codes.view(torch.int8).permute(0, 2, 1, 3)[~mine] = bad
        scale[~mine.any(1)] = math.nan


def to(pages, device):
    return type(pages)(*(t.to(device) for t in pages))
