"""A paged cache held in 8 bits: half the bytes of a 16-bit one, in the memory and on every read.

A pool of pages holds codes of K and V, ``[pages, Hkv, page, D]`` e4m3 or 8-bit integers, and one
fp32 scale a (page, KV head) of each: value = scale * code. A page table ``[B, M]`` int32 maps a
sequence's token t to row ``t % page`` of page ``page_table[b, t // page]``; entries outside the
pool (-1) hold no keys. The operators: ``append_quantized`` (new tokens, in place),
``quantized_attention`` (all keys), ``quantized_read`` (a selection's lists, what ``paged_read`` is for
16-bit pools), ``move_pages`` (copies). ``QuantizedCache`` keeps the books on the host: which
pages a sequence holds, which are shared, which are free. No reference counterpart: the reference
has a slot table in its walk and no allocator (``paged.py``).

    cache = QuantizedCache(places=64, pages=8192, kv_heads=8, head_dim=128)
    cache.append([0], k_prompt, v_prompt)            # [1, T, Hkv, D]
    child = cache.fork(0)                            # shares every page until one of them writes
    out = cache.step([0, child], q, k, v)            # append, then attend
    cache.free([child])
"""

from __future__ import annotations

import heapq
from typing import NamedTuple

import numpy as np
import torch

from . import _lib


class QuantizedPages(NamedTuple):
    k: torch.Tensor  # [pages, Hkv, page, D] float8_e4m3fn or int8; page 16, 32, 64 or 128, D 64 or 128
    v: torch.Tensor  # like k
    k_scale: torch.Tensor  # [pages, Hkv] fp32
    v_scale: torch.Tensor  # [pages, Hkv] fp32

    @classmethod
    def new(cls, pages: int, kv_heads: int, page: int, head_dim: int, dtype=torch.float8_e4m3fn, device="cuda"):
        """A pool of zeros."""
        def codes():
            return torch.zeros(pages, kv_heads, page, head_dim, dtype=torch.int8, device=device).view(dtype)

        def scales():
            return torch.ones(pages, kv_heads, dtype=torch.float32, device=device)

        return cls(codes(), codes(), scales(), scales())


def append_quantized(pages: QuantizedPages, k, v, page_table, lengths, counts=None) -> None:
    """Write the last Tq tokens of every sequence into its pages, in place.

    k, v [B, Tq, Hkv, D] fp32, fp16 or bf16 (strided views as in ``shared_prefix_attention``); ``lengths``
    [B] count the tokens that a sequence then holds: row i is token ``lengths[b] - Tq + i``, and
    rows before token 0 are padding (a sequence of length 0 gets nothing), and so are all but the last
    ``counts[b]`` rows where counts [B] are given. Tokens on pages that
    the table does not map are dropped. A page's scale is the smallest power of two, at least 2^-60,
    with which its largest new magnitude fits the codes (448, 127), or the scale it has, if older
    tokens of the page need more; when it grows, the page's older codes are rounded to it. Codes are rounded to
    the nearest, ties to even. New values must be finite. Pages that a call writes belong to one sequence: with the
    same page in two rows its content is undefined. What a page holds behind the last token stays."""
    _lib.torch_ops().append_quantized(k, v, pages.k, pages.v, pages.k_scale, pages.v_scale, page_table, lengths,
                                      counts)
    _lib.after_call(k.device, "append_quantized")


def quantized_attention(q, pages: QuantizedPages, page_table, lengths, scale=None, return_lse: bool = False):
    """Dense attention of q's rows over the sequences' pages.

    q [B, Tq, Hq, D] fp16 or bf16; sequence b holds ``lengths[b]`` tokens, the call's Tq new ones among
    them (append first). Row i sees the tokens ``j < lengths[b] - Tq + i + 1`` on pages that the table
    maps; a row that sees none reads as zeros (log-sum-exp -inf), whatever q holds there; one of q that is
    not finite and sees a key is NaN. What pages hold behind a sequence's last token is never used; what
    a row of the call sees must be finite, its scales positive, the value scales within 2^100 of each
    other (they count as 2^-60 at least). ``scale``, positive, defaults to ``D ** -0.5``. The weights are
    rounded to 16 bits for their product with the codes; sums, joins and log-sum-exp are fp32. Output
    like q, contiguous; with ``return_lse`` also the natural log-sum-exp of every row's scaled logits,
    fp32 [B, Tq, Hq]."""
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    ops = _lib.torch_ops()
    fn = ops.quantized_attention_lse if return_lse else ops.quantized_attention
    out = fn(q, pages.k, pages.v, pages.k_scale, pages.v_scale, page_table, lengths, scale)
    _lib.after_call(q.device, "quantized_attention")
    return out


def quantized_read(q, pages: QuantizedPages, page_table, lengths, lists, counts, rows=None, scale=None):
    """The sparse read over the pages: query row r attends to the listed positions of a sequence.

    q [R, 1, Hq, D] fp16 or bf16, a list a row (``flat_select``, ``tree_select``; a tile's shared
    lists are ``sparse_prefill``'s); ``lists`` [R, W] int32 positions in any order, ``counts`` [R] how many
    of a row's entries count; row r reads sequence ``rows[r]`` of the table (r itself when None). Positions
    outside [0, lengths[rows[r]]), on unmapped pages, and rows outside the table are skipped;
    duplicates count per occurrence; a row without keys reads as zeros. Otherwise as ``quantized_attention``."""
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    out = _lib.torch_ops().quantized_read(q, pages.k, pages.v, pages.k_scale, pages.v_scale, page_table, lengths,
                                          lists, counts, rows, scale)
    _lib.after_call(q.device, "quantized_read")
    return out


def move_pages(pages: QuantizedPages, src, dst) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` (codes and scales, every head), all in one launch.

    src, dst [n] int32; pairs with an index outside the pool are skipped. No page may be written twice
    or both read and written: its content is undefined then."""
    _lib.torch_ops().move_pages(pages.k, pages.v, pages.k_scale, pages.v_scale, src, dst)
    _lib.after_call(pages.k.device, "move_pages")


class QuantizedCache:
    """The caches of a serving batch over one pool of 8-bit pages.

    ``places`` sequences at most, ``pages`` pages of ``page`` tokens. Which pages a sequence holds is known
    on the host, so nothing asks the device; a call uploads the lengths and the table rows it
    needs (so the methods are not for stream capture; the operators are). A refused call (ValueError) leaves
    the cache as it was."""

    def __init__(self, places: int, pages: int, kv_heads: int, head_dim: int, page: int = 64,
                 dtype=torch.float8_e4m3fn, device="cuda"):
        if not 1 <= places <= 65535 or pages < 1:
            raise ValueError(f"a cache has pages and 1 to 65535 places, got {pages} and {places}")
        if page not in (16, 32, 64, 128) or head_dim not in (64, 128) or kv_heads < 1:
            raise ValueError(f"pages of 16, 32, 64 or 128 tokens and heads of 64 or 128, got {page} and {head_dim}")
        if dtype not in (torch.float8_e4m3fn, torch.int8):
            raise ValueError(f"codes are float8_e4m3fn or int8, got {dtype}")
        if kv_heads > 65535 or pages * kv_heads * page > (1 << 31) - 1:  # the operators' limits
            raise ValueError(f"at most 65535 heads and fewer than 2^31 (page, head, token) rows, got {kv_heads} heads, "
                             f"{pages} pages of {page}")
        self.pages = QuantizedPages.new(pages, kv_heads, page, head_dim, dtype, device)
        self.page = page
        self.lengths = [0] * places  # tokens of every place
        self._held: list[list[int]] = [[] for _ in range(places)]  # their pages
        self._refs = [0] * pages
        self._free = list(range(pages))  # a heap: the lowest page first

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _places(self, places, what):
        places = [int(p) for p in places]
        if any(p < 0 or p >= len(self._held) for p in places):
            raise ValueError(f"{what}: places in [0, {len(self._held)}), got {places}")
        return places

    def _check_rows(self, what, n, Tq, *tensors):
        for t in tensors:
            if t.dim() != 4 or t.shape[0] != n or t.shape[1] != Tq:
                raise ValueError(f"{what}: [{n}, {Tq}, heads, {self.pages.k.shape[3]}], got {list(t.shape)}")
            if t.device != self.pages.k.device:
                raise ValueError(f"{what}: tensors on {self.pages.k.device}, got {t.device}")

    def _check_new(self, what, n, k, v):
        Hkv, D = self.pages.k.shape[1], self.pages.k.shape[3]
        self._check_rows(what, n, k.shape[1] if k.dim() == 4 else -1, k, v)
        if k.shape[2:] != (Hkv, D) or v.shape != k.shape:
            raise ValueError(f"{what}: keys and values are [{n}, Tq, {Hkv}, {D}], got {list(k.shape)}, {list(v.shape)}")
        if k.dtype not in _lib.DTYPE_CODE or v.dtype != k.dtype:
            raise ValueError(f"{what}: fp32, fp16 or bf16 keys and values of one type, got {k.dtype}, {v.dtype}")

    def _staged(self, n):
        """n int32 on the host, pinned where the pages are on a GPU: a copy from pageable memory would wait for all
        that the stream holds. Torch keeps pinned memory until the copies from it have run."""
        return torch.empty(n, dtype=torch.int32, device="cpu", pin_memory=self.pages.k.is_cuda)

    def _upload(self, places, counts=()):
        """(page table, lengths, counts) of the places on the device, in one copy."""
        n, M = len(places), max([len(self._held[p]) for p in places], default=0)
        staged = self._staged(n * (M + 2))
        host = staged.numpy()
        host[:] = -1
        host[:n] = [self.lengths[p] for p in places]
        host[n:n + len(counts)] = counts
        table = host[2 * n:].reshape(n, M)
        for i, p in enumerate(places):
            table[i, :len(self._held[p])] = self._held[p]
        dev = staged.to(self.pages.k.device, non_blocking=True)
        return dev[2 * n:].view(n, M), dev[:n], dev[n:2 * n]

    def _grow(self, places, counts, Tq):
        """Pages for the new tokens; a shared page that they would write becomes the sequence's own copy."""
        if len(set(places)) != len(places):
            raise ValueError(f"append: a place once, got {places}")
        counts = [Tq] * len(places) if counts is None else [int(c) for c in counts]
        if len(counts) != len(places) or any(c < 0 or c > Tq for c in counts):
            raise ValueError(f"append: one count in [0, {Tq}] a place, got {counts}")
        if any(self.lengths[p] + c > 1 << 30 for p, c in zip(places, counts)):
            raise ValueError("append: a sequence holds at most 2^30 tokens")
        need, refs = 0, {}
        copies = []
        for p, c in zip(places, counts):
            length, held = self.lengths[p], self._held[p]
            need += -(-(length + c) // self.page) - len(held)
            if c and length % self.page:
                last = held[-1]
                if refs.setdefault(last, self._refs[last]) > 1:
                    refs[last] -= 1
                    copies.append(p)
        if need + len(copies) > len(self._free):
            raise ValueError(f"append: {need + len(copies)} pages needed, {len(self._free)} free")
        src, dst = [], []
        for p in copies:
            new = heapq.heappop(self._free)
            src.append(self._held[p][-1])
            dst.append(new)
            self._refs[src[-1]] -= 1
            self._refs[new] = 1
            self._held[p][-1] = new
        for p, c in zip(places, counts):
            self.lengths[p] += c
            for _ in range(-(-self.lengths[p] // self.page) - len(self._held[p])):
                new = heapq.heappop(self._free)
                self._refs[new] = 1
                self._held[p].append(new)
        self._move(src, dst)
        return counts

    def _move(self, src, dst):
        if src:
            staged = self._staged(2 * len(src))
            staged.numpy()[:] = src + dst
            ids = staged.to(self.pages.k.device, non_blocking=True)
            move_pages(self.pages, ids[:len(src)], ids[len(src):])

    def append(self, places, k, v, counts=None) -> None:
        """Append k, v [n, Tq, Hkv, D] to the n places; of place i's rows the last ``counts[i]`` (all of them
        when None), the others are padding. ValueError when the pages run out."""
        places = self._places(places, "append")
        self._check_new("append", len(places), k, v)
        counts = self._grow(places, counts, k.shape[1])
        if places:
            append_quantized(self.pages, k, v, *self._upload(places, counts))

    def attend(self, places, q, scale=None):
        """``quantized_attention`` of q [n, Tq, Hq, D], the places' last Tq tokens, over what they hold."""
        places = self._places(places, "attend")
        self._check_rows("attend", len(places), q.shape[1] if q.dim() == 4 else -1, q)
        table, lengths, _ = self._upload(places)
        return quantized_attention(q, self.pages, table, lengths, scale)

    def step(self, places, q, k, v, scale=None):
        """Append, then attend, with one upload. Output like q."""
        places = self._places(places, "step")
        self._check_new("step", len(places), k, v)
        self._check_rows("step", len(places), k.shape[1], q)
        Hkv, D = self.pages.k.shape[1], self.pages.k.shape[3]
        if q.dtype not in (torch.float16, torch.bfloat16) or q.shape[3] != D or q.shape[2] % Hkv or q.shape[2] < Hkv:
            raise ValueError(f"step: q is fp16 or bf16 [n, Tq, a multiple of {Hkv}, {D}], got {q.dtype} {list(q.shape)}")
        with np.errstate(over="ignore", under="ignore"):  # as the operator takes it: it refuses after the append
            scale_log2 = np.float32(D ** -0.5 if scale is None else float(scale)) * np.float32(1.4426950408889634)
        if not 0 < scale_log2 < np.inf:
            raise ValueError(f"step: the scale must be positive, and with log2(e) within fp32, got {scale}")
        n, Tq = q.shape[:2]
        M = max([-(-(self.lengths[p] + Tq) // self.page) for p in places], default=0)
        if _lib.lib().lsa_quantized_scratch(n, Tq, q.shape[2], Hkv, D, M * self.page, 0) < 0:
            raise ValueError(f"step: sizes out of range, q {list(q.shape)}")
        self._grow(places, None, Tq)
        table, lengths, _ = self._upload(places)
        if places:
            append_quantized(self.pages, k, v, table, lengths)
        return quantized_attention(q, self.pages, table, lengths, scale)

    def read(self, places, q, lists, counts, scale=None):
        """``quantized_read`` of q [n, 1, Hq, D]: row i attends to the positions ``lists[i, :counts[i]]`` of place i."""
        places = self._places(places, "read")
        self._check_rows("read", len(places), 1, q)
        table, lengths, _ = self._upload(places)
        return quantized_read(q, self.pages, table, lengths, lists, counts, None, scale)

    def fork(self, place: int) -> int:
        """A free place that holds what ``place`` holds, on the same pages; whichever of the two writes to
        a shared page first takes a copy of it then. ``place`` holds something: an empty one's fork would be
        free still, for the next fork to take."""
        (place,) = self._places([place], "fork")
        if not self._held[place]:
            raise ValueError(f"fork: place {place} is empty")
        free = next((i for i, held in enumerate(self._held) if not held and i != place), None)
        if free is None:
            raise ValueError("fork: no free place")
        self._held[free] = list(self._held[place])
        self.lengths[free] = self.lengths[place]
        for p in self._held[free]:
            self._refs[p] += 1
        return free

    def free(self, places) -> None:
        """Empty the places; pages that no other place holds are free again."""
        for p in self._places(places, "free"):
            for page in self._held[p]:
                self._refs[page] -= 1
                if self._refs[page] == 0:
                    heapq.heappush(self._free, page)
            self._held[p], self.lengths[p] = [], 0

    def compact(self) -> int:
        """Move the pages in use to the front of the pool, in one launch; returns how many there are."""
        used = len(self._refs) - len(self._free)
        src = [p for p in range(used, len(self._refs)) if self._refs[p]]
        dst = [p for p in range(used) if not self._refs[p]]
        to = dict(zip(src, dst))
        for s, d in to.items():
            self._refs[d], self._refs[s] = self._refs[s], 0
        self._held = [[to.get(p, p) for p in held] for held in self._held]
        self._free = list(range(used, len(self._refs)))
        self._move(src, dst)
        return used
