"""The 8-bit paged cache on a B200 against its definitions in 64 bits (quantized_forms.py has the tolerances)."""

import math

import pytest
import torch

import quantized_forms as F

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def close(got, want, off, what=""):
    got, most = got.cpu(), torch.finfo(got.dtype).max
    got = got.double()
    bad = ~((got - want).abs() <= off) & ~(got == want)
    # a value that rounds past the type's largest is an infinity of its sign, by the definition of rounding
    bad &= ~(got.isinf() & (got.sign() == want.sign()) & (want.abs() + off >= most))
    assert not bad.any(), (what, int(bad.sum()), float(((got - want).abs() / off)[bad].max()))


def same(got, want):
    """The same values (a zero may have either sign) and scales."""
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and torch.equal(a.cpu().float(), b.cpu().float())


def attend_case(lsa, seed, lengths, Tq, Hq, Hkv, D, page, code, dtype, spread=2.0, scale=None):
    g = torch.Generator().manual_seed(seed)
    table, n = F.paged(g, lengths, page)
    pages = F.pool(g, n, Hkv, page, D, code, spread)
    F.poison(pages, table, lengths)
    q = torch.randn(len(lengths), Tq, Hq, D, generator=g).to(dtype)
    ln = torch.tensor(lengths, dtype=torch.int32)
    want, lse, off, lse_off = F.attention(q, pages, table, ln, scale)
    got, got_lse = lsa.quantized_attention(q.cuda(), F.to(pages, "cuda"), table.cuda(), ln.cuda(), scale, return_lse=True)
    assert got.dtype == dtype and got.shape == q.shape and got_lse.shape == lse.shape
    close(got, want, off, "out")
    close(got_lse, lse, lse_off + 2.0 ** -22, "lse")
    only = lsa.quantized_attention(q.cuda(), F.to(pages, "cuda"), table.cuda(), ln.cuda(), scale)
    assert torch.equal(only, got)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths,Tq,Hq,Hkv,page", [
    ([1], 1, 1, 1, 16),
    ([0, 5, 16, 17, 33], 1, 8, 2, 16),
    ([200, 64, 63, 65], 1, 12, 4, 64),
    ([1000, 0, 257], 3, 8, 1, 32),
    ([127, 128, 129, 2], 5, 3, 3, 128),
])
def test_attention_decode(lsa, code, dtype, D, lengths, Tq, Hq, Hkv, page):
    attend_case(lsa, 1, lengths, Tq, Hq, Hkv, D, page, code, dtype)


@pytest.mark.parametrize("code,dtype,D,page", [("e4m3", BF, 128, 64), ("int8", HF, 64, 16), ("e4m3", HF, 128, 128)])
def test_attention_long(lsa, code, dtype, D, page):
    """Long enough that a sequence's keys are split over many CTAs, beside a short one."""
    attend_case(lsa, 2, [9001, 3], 1, 8, 2, D, page, code, dtype)


@pytest.mark.parametrize("Tq", [6, 33, 100, 200])
@pytest.mark.parametrize("code,dtype,D,page,Hq,Hkv", [
    ("e4m3", BF, 128, 64, 4, 1), ("int8", HF, 64, 16, 8, 4), ("e4m3", HF, 128, 32, 3, 1), ("int8", BF, 128, 128, 2, 2)])
def test_attention_chunks(lsa, Tq, code, dtype, D, page, Hq, Hkv):
    """Prompts of several tokens: lengths below Tq (rows that see nothing), equal to it, and beyond."""
    attend_case(lsa, 3, [Tq + 777, Tq, Tq // 2, 0, Tq + 1], Tq, Hq, Hkv, D, page, code, dtype)


# What the tensor-core kernel takes: more rows x keys than the few-row kernel is faster on.
@pytest.mark.parametrize("Tq,Hq,Hkv", [(9, 32, 8), (16, 32, 8), (13, 48, 8), (31, 32, 8), (64, 16, 4), (65, 24, 8)],
                         ids=["36rows", "64rows", "78rows", "124rows", "two halves", "odd group"])
@pytest.mark.parametrize("code,dtype,D,page", [("e4m3", BF, 128, 64), ("int8", HF, 64, 16), ("e4m3", HF, 64, 128),
                                               ("int8", BF, 128, 32)])
def test_attention_tiles(lsa, Tq, Hq, Hkv, code, dtype, D, page):
    """Ragged batches: no key, fewer keys than rows, one chunk, its border, several; two streams with one to four
    warps of rows, both halves."""
    g = torch.Generator().manual_seed(Tq)
    lengths = [0, 1, Tq - 1, Tq, 127, 128, 129, 255, 256, 257, 383, 1100, 1152] + torch.randint(1, 1152, (9,), generator=g).tolist()
    attend_case(lsa, 20, lengths, Tq, Hq, Hkv, D, page, code, dtype)


def test_attention_tiles_long(lsa):
    """A long sequence's tiles split over many CTAs beside short ones; scales far apart; holes in the table."""
    attend_case(lsa, 21, [9003, 70, 4096], 70, 16, 2, 128, 64, "e4m3", BF)
    attend_case(lsa, 22, [3000] * 5, 40, 16, 8, 128, 16, "e4m3", HF, spread=60.0, scale=1e-6)
    g = torch.Generator().manual_seed(23)
    lengths = [1500] * 12
    for Tq in (10, 70):
        table, n = F.paged(g, lengths, 32)
        table[:, 3::5], table[2], table[5, 1:] = -1, 1 << 30, -1
        pages = F.pool(g, n, 8, 32, 64, "int8")
        F.poison(pages, table, lengths)
        q = torch.randn(12, Tq, 32, 64, generator=g).to(BF)
        q[3, Tq - 1, 7, 5] = math.nan
        ln = torch.tensor(lengths)
        want, _, off, _ = F.attention(q, pages, table, ln)
        got = lsa.quantized_attention(q.cuda(), F.to(pages, "cuda"), table.cuda(), ln.cuda()).cpu()
        assert got[3, Tq - 1, 7].isnan().all()
        keep = torch.ones(12, Tq, 32, dtype=torch.bool)
        keep[3, Tq - 1, 7] = False
        close(got[keep], want[keep], off[keep])


@pytest.mark.parametrize("Tq", [1, 40])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_attention_scales_far_apart(lsa, Tq, dtype):
    """Value and key scales that differ from page to page by up to 2^60."""
    attend_case(lsa, 4, [700, Tq + 90], Tq, 4, 2, 128, 16, "e4m3", dtype, spread=60.0, scale=1e-6)


@pytest.mark.parametrize("Tq", [1, 40])
def test_attention_large_logits(lsa, Tq):
    attend_case(lsa, 5, [500, Tq + 300], Tq, 4, 2, 128, 64, "e4m3", BF, scale=3.0)


@pytest.mark.parametrize("Tq", [1, 40])
def test_attention_unmapped_pages_and_strides(lsa, Tq):
    """Holes in the table, indices outside the pool, a table that is a slice, q as a slice of a projection, int64."""
    g = torch.Generator().manual_seed(6)
    lengths = [Tq + 300, Tq + 100]
    table, n = F.paged(g, lengths, 32)
    table[0, 2], table[0, 4], table[1, 0] = -1, 1 << 30, -(1 << 31)
    pages = F.pool(g, n, 2, 32, 128, "e4m3")
    q = torch.randn(2, Tq, 6, 128, generator=g).to(BF)
    ln = torch.tensor(lengths)
    want, _, off, _ = F.attention(q, pages, table, ln)
    wide = torch.full((2, table.shape[1] + 5), 7, dtype=torch.int32)
    wide[:, 2:2 + table.shape[1]] = table
    qkv = torch.randn(2, Tq, 10, 128).to(BF).cuda()
    qkv[:, :, 1:7] = q.cuda()
    dev = F.to(pages, "cuda")
    for t in (wide.cuda()[:, 2:2 + table.shape[1]], table.long().cuda()):
        close(lsa.quantized_attention(qkv[:, :, 1:7], dev, t, ln.cuda()), want, off)


@pytest.mark.parametrize("Tq", [1, 40])
def test_attention_row_of_nan_stays_its_own(lsa, Tq):
    g = torch.Generator().manual_seed(7)
    lengths = [Tq + 50, Tq + 200]
    table, n = F.paged(g, lengths, 64)
    pages = F.pool(g, n, 1, 64, 128, "e4m3")
    q = torch.randn(2, Tq, 4, 128, generator=g).to(BF)
    ln = torch.tensor(lengths, dtype=torch.int32)
    want, _, off, _ = F.attention(q, pages, table, ln)
    q[1, 0, 2, 5], q[0, Tq - 1, 1, 0] = math.nan, math.inf
    got = lsa.quantized_attention(q.cuda(), F.to(pages, "cuda"), table.cuda(), ln.cuda()).cpu()
    assert got[1, 0, 2].isnan().all() and got[0, Tq - 1, 1].isnan().any()
    keep = torch.ones(2, Tq, 4, dtype=torch.bool)
    keep[1, 0, 2] = keep[0, Tq - 1, 1] = False
    close(got[keep], want[keep], off[keep])


def test_attention_beyond_32_bits(lsa):
    """Pages whose codes lie past 2^32 bytes of the pool."""
    n, Hkv, page, D = 70000, 8, 64, 128
    g = torch.Generator().manual_seed(8)
    lengths = [150, 64]
    table, _ = F.paged(g, lengths, page, 0)
    small = F.pool(g, 4, Hkv, page, D, "e4m3")
    far = torch.tensor([n - 1, n - 2, 66000, 3])
    big = lsa.QuantizedPages.new(n, Hkv, page, D)
    for b, s in zip(big, small):
        b = b.view(torch.int8) if b.element_size() == 1 else b
        s = s.view(torch.int8) if s.element_size() == 1 else s
        b[far.cuda()] = s.cuda()
    q = torch.randn(2, 1, 16, D, generator=g).to(BF)
    ln = torch.tensor(lengths, dtype=torch.int32)
    want, _, off, _ = F.attention(q, small, table, ln)
    moved = torch.where(table >= 0, far.to(torch.int32)[table.clamp(min=0)], table)
    close(lsa.quantized_attention(q.cuda(), big, moved.cuda(), ln.cuda()), want, off)
    qc = torch.randn(2, 40, 16, D, generator=g).to(BF)
    want, _, off, _ = F.attention(qc, small, table, ln)
    close(lsa.quantized_attention(qc.cuda(), big, moved.cuda(), ln.cuda()), want, off)
    k = torch.randn(2, 2, Hkv, D, generator=g)
    v = torch.randn(2, 2, Hkv, D, generator=g)
    F.append(small, k, v, table, ln)
    lsa.append_quantized(big, k.cuda(), v.cuda(), moved.cuda(), ln.cuda())
    same([b.view(torch.int8)[far.cuda()].view(b.dtype) if b.element_size() == 1 else b[far.cuda()] for b in big], small)
    lsa.move_pages(big, torch.tensor([n - 1, 66000]).cuda(), torch.tensor([5, n - 7]).cuda())
    same([b.view(torch.int8)[[5, n - 7]].view(b.dtype) if b.element_size() == 1 else b[[5, n - 7]] for b in big],
         [s.view(torch.int8)[[0, 2]].view(s.dtype) if s.element_size() == 1 else s[[0, 2]] for s in small])


@pytest.mark.parametrize("Tq", [12, 24, 31])
def test_attention_many_sequences(lsa, Tq):
    """More (sequence, KV head) pairs than the split tiles' rounds: nothing is kept for them beside the output."""
    g = torch.Generator().manual_seed(Tq)
    lengths = torch.randint(0, 200, (1201,), generator=g).tolist()
    attend_case(lsa, 40 + Tq, lengths, Tq, 4, 1, 64, 32, "e4m3", BF)
    from lsa_b200 import _lib

    assert _lib.lib().lsa_quantized_scratch(1 << 14, Tq, 4, 1, 64, 224, 0) <= 157 << 20


@pytest.mark.parametrize("shape", [(0, 1, 3), (2, 0, 3), (2, 1, 0)])
def test_attention_empty(lsa, shape):
    B, Tq, M = shape
    pages = lsa.QuantizedPages.new(4, 2, 16, 64)
    q = torch.randn(B, Tq, 4, 64, device="cuda").to(BF)
    table = torch.zeros(B, M, dtype=torch.int32, device="cuda")
    ln = torch.full((B,), 20, dtype=torch.int32, device="cuda")
    out, lse = lsa.quantized_attention(q, pages, table, ln, return_lse=True)
    assert out.shape == q.shape and bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("M", [0, 1])
def test_attention_many_rows_on_no_key(lsa, M):
    """Rows of a long call whose table maps nothing, or one page behind almost all of them."""
    pages = lsa.QuantizedPages.new(4, 8, 16, 64)
    q = torch.zeros(1, 1 << 15, 64, 64, device="cuda", dtype=BF)
    table = torch.zeros(1, M, dtype=torch.int32, device="cuda")
    if M:
        ones = torch.ones(1, 5, 8, 64, device="cuda")
        lsa.append_quantized(pages, ones, ones, table, torch.tensor([5]).cuda())
    out, lse = lsa.quantized_attention(q, pages, table, torch.tensor([5]).cuda(), return_lse=True)
    seen = 5 * M
    assert bool((out[:, :(1 << 15) - seen] == 0).all()) and bool((lse[:, :(1 << 15) - seen] == -math.inf).all())
    if M:  # equal logits of zero: the values' mean, and the number of keys
        assert bool((out[:, -seen:] == 1).all())
        want = torch.arange(1, 6, device="cuda").log()[None, :, None].expand(1, 5, 64)
        # log2 of a sum of up to 2^20.4, an ulp off, and two more roundings below it
        assert bool(((lse[:, -seen:] - want).abs() <= 2.0 ** -18).all())


@pytest.mark.parametrize("Tq,Hq,Hkv", [(1, 160, 1), (2, 33, 1), (3, 130, 1), (9, 21, 3)])
def test_attention_head_groups(lsa, Tq, Hq, Hkv):
    """Groups of odd sizes, and of more heads than a row tile of the tensor cores holds."""
    attend_case(lsa, 18, [300, Tq, 40], Tq, Hq, Hkv, 64, 32, "e4m3", BF)


@pytest.mark.parametrize("Tq", [1, 40])
def test_attention_of_an_empty_pool(lsa, Tq):
    pages = lsa.QuantizedPages.new(0, 2, 16, 64)
    q = torch.randn(2, Tq, 4, 64, device="cuda").to(BF)
    table, ln = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.tensor([40, 5], device="cuda")
    out, lse = lsa.quantized_attention(q, pages, table, ln, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    lists = torch.zeros(2, 7, dtype=torch.int32, device="cuda")
    assert bool((lsa.quantized_read(q[:, :1], pages, table, ln, lists, ln) == 0).all())
    lsa.append_quantized(pages, q[:, :, :2], q[:, :, :2], table, ln)
    lsa.move_pages(pages, lists[0], lists[1])
    none = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    some = lsa.QuantizedPages.new(3, 2, 16, 64)
    assert bool((lsa.quantized_read(q[:, :1], some, table, ln, none, ln) == 0).all())


@pytest.fixture()
def wait_limit():
    """Sets the limit of the tensor-core kernels' waits (ns); the default again afterwards."""
    from lsa_b200 import _lib

    _lib.torch_ops()
    yield lambda ns: _lib.check(_lib.lib().lsa_shared_prefix_wait_limit(ns), "wait limit")
    assert _lib.lib().lsa_shared_prefix_wait_limit(-1) == _lib.OK


@pytest.mark.parametrize("code,D,page,B,Tq,Hq,Hkv,T", [
    ("e4m3", 128, 64, 20, 16, 32, 4, 3000),  # two streams, split
    ("int8", 64, 16, 24, 40, 8, 4, 700),
    ("e4m3", 128, 128, 40, 64, 32, 4, 900),  # both halves, whole tiles and split ones
    ("int8", 64, 32, 12, 257, 6, 2, 257),
])
def test_expired_waits_leave_with_their_copies_landed(lsa, wait_limit, code, D, page, B, Tq, Hq, Hkv, T):
    """Every role gives up at its first wait, with the first copies in flight. The call reports it, and calls after it,
    on the same SMs, answer as before."""
    g = torch.Generator().manual_seed(19)
    lengths = torch.randint(min(Tq, T), T + 1, (B,), generator=g).tolist()
    table, n = F.paged(g, lengths, page)
    pages = F.to(F.pool(g, n, Hkv, page, D, code), "cuda")
    q = torch.randn(B, Tq, Hq, D, generator=g).to(BF).cuda()
    table, ln = table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()
    want = lsa.quantized_attention(q, pages, table, ln)
    for _ in range(3):
        wait_limit(0)
        with pytest.raises(RuntimeError, match="bounded device wait expired"):
            lsa.quantized_attention(q, pages, table, ln)
            lsa.check_status()  # without the checked mode
        wait_limit(-1)
        assert torch.equal(lsa.quantized_attention(q, pages, table, ln), want)
    lsa.check_status()


# ------------------------------------------------------------------ the read


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype,D,page,Hq,Hkv,W", [(BF, 128, 64, 8, 2, 300), (HF, 64, 16, 8, 1, 1), (BF, 64, 128, 3, 3, 70),
                                                   (HF, 128, 32, 20, 1, 2116)])
def test_read(lsa, code, dtype, D, page, Hq, Hkv, W):
    g = torch.Generator().manual_seed(9)
    lengths = [500, 0, 33, 4000]
    table, n = F.paged(g, lengths, page)
    table[3, 1] = -1
    pages = F.pool(g, n, Hkv, page, D, code)
    F.poison(pages, table, lengths)
    R = 6
    rows = torch.tensor([3, 0, 0, 2, 1, 9], dtype=torch.int32)
    lists = torch.randint(-3, 4100, (R, W), generator=g, dtype=torch.int32)
    lists[1] = torch.randint(0, 500, (W,), generator=g, dtype=torch.int32)  # with duplicates
    lists[2, :] = 499
    lists[3, ::2] = 1 << 30
    counts = torch.tensor([W, W, W, W, W, W], dtype=torch.int32)
    counts[0], counts[2] = W + 9, max(1, W // 2)
    q = torch.randn(R, 1, Hq, D, generator=g).to(dtype)
    ln = torch.tensor(lengths, dtype=torch.int32)
    want, off = F.read(q, pages, table, ln, lists, counts, rows)
    dev = F.to(pages, "cuda")
    got = lsa.quantized_read(q.cuda(), dev, table.cuda(), ln.cuda(), lists.cuda(), counts.cuda(), rows.cuda())
    close(got, want, off)
    assert bool((got[4] == 0).all()) and bool((got[5] == 0).all())
    counts.zero_()
    got = lsa.quantized_read(q.cuda(), dev, table.cuda(), ln.cuda(), lists.cuda(), counts.cuda(), rows.cuda())
    assert bool((got == 0).all())
    counts[:4] = W
    rows = torch.arange(4, dtype=torch.int32)
    want, off = F.read(q[:4], pages, table, ln, lists[:4], counts[:4], rows)
    close(lsa.quantized_read(q[:4].cuda(), dev, table.cuda(), ln.cuda(), lists[:4].cuda(), counts[:4].cuda()), want, off)


def test_read_of_a_selection_equals_the_16_bit_paged_read(lsa):
    """The framework's own selection, read over the 8-bit pages and, their values as fp16, over a 16-bit pool."""
    from lsa_b200 import paged

    g = torch.Generator().manual_seed(10)
    T, Hkv, Hq, D, page = 4096, 2, 8, 128, 64
    table, n = F.paged(g, [T], page)
    pages = F.pool(g, n, Hkv, page, D, "e4m3", spread=0.0)
    for s in (pages.k_scale, pages.v_scale):
        s.copy_(torch.exp2(torch.log2(s).round()))  # values that are halves exactly
    ids, key, val = F.keys(pages, table[0], torch.arange(T))
    k, v = key.half().cuda(), val.half().cuda()
    assert torch.equal(k.double().cpu(), key) and torch.equal(v.double().cpu(), val)
    q = torch.randn(1, Hq, D, generator=g).half().cuda()
    iq, ik = lsa.make_index_space(torch.cat([q.expand(T - 1, Hq, D), q])[None], k[None])
    cfg = lsa.PortConfig(cluster_block_size=512, pool_size=4, bucket_size=64, bucket_cap=128, top_p=4, top_k=256,
                         window_size=64, sink_size=4)
    buckets = lsa.build_buckets_gpu(ik, cfg)
    pos = torch.tensor([T - 1], device="cuda")
    lists, counts = lsa.flat_select(iq[-1:], pos, buckets, cfg)
    kv = paged.pack_paged(k[None], v[None], [T])
    rows = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = paged.paged_read(q[:, None], kv, lists, counts, rows)
    ln = torch.tensor([T], dtype=torch.int32)
    got = lsa.quantized_read(q[:, None], F.to(pages, "cuda"), table.cuda(), ln.cuda(), lists, counts, rows)
    exact, off = F.read(q[:, None].cpu(), pages, table, ln, lists.cpu(), counts.cpu(), rows.cpu())
    close(got, exact, off)
    assert (got - want).abs().max() <= 2 * off.max() + 2e-3


# ------------------------------------------------------------------ append, moves


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float32, HF, BF])
@pytest.mark.parametrize("D,page,Tq,lengths", [
    (128, 64, 1, [1, 64, 65, 0, 100]),
    (64, 16, 1, [33, 32, 17]),
    (128, 16, 4, [4, 2, 20, 0, 18]),
    (64, 128, 5, [130, 128, 3, 200]),
    (128, 32, 77, [77, 300, 50, 0, 78]),
    (128, 128, 300, [300, 500, 128]),
])
def test_append(lsa, code, dtype, D, page, Tq, lengths):
    g = torch.Generator().manual_seed(11)
    Hkv = 3
    table, n = F.paged(g, lengths, page)
    pages = F.pool(g, n, Hkv, page, D, code)
    k, v = (torch.randn(len(lengths), Tq, Hkv, D, generator=g).to(dtype) for _ in range(2))
    k[0] *= 37.0  # a page's scale grows
    v[-1] *= 1e-3  # and stays
    if dtype == torch.float32:
        k[-1] *= 1e-25  # below the smallest scale
    ln = torch.tensor(lengths, dtype=torch.int32)
    dev = F.to(pages, "cuda")
    F.append(pages, k, v, table, ln)
    lsa.append_quantized(dev, k.cuda(), v.cuda(), table.cuda(), ln.cuda())
    same(dev, pages)
    lsa.append_quantized(dev, k.cuda(), v.cuda(), table.cuda(), ln.cuda())  # again: as it was
    same(dev, pages)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_append_grows_pages_token_by_token(lsa, code):
    """Every token larger than the ones before it: the page's older codes are rounded to each new scale in turn."""
    g = torch.Generator().manual_seed(12)
    table, n = F.paged(g, [40], 16)
    pages = F.pool(g, n, 2, 16, 64, code)
    dev = F.to(pages, "cuda")
    for t in range(40):
        k, v = (torch.randn(1, 1, 2, 64, generator=g) * 1.5 ** t for _ in range(2))
        ln = torch.tensor([t + 1], dtype=torch.int32)
        F.append(pages, k, v, table, ln)
        lsa.append_quantized(dev, k.cuda(), v.cuda(), table.cuda(), ln.cuda())
    same(dev, pages)


def test_append_padding_counts_and_holes(lsa):
    """NaN in padding rows stays out; rows on unmapped pages, or behind the table, are dropped; strided k and v."""
    g = torch.Generator().manual_seed(13)
    lengths, page, Tq = [50, 30, 200, 10, 64], 32, 20
    table, n = F.paged(g, lengths, page)
    table[1, 0] = -1
    table[2, 6] = n + 5
    table = table[:, :6].contiguous()  # sequence 2 holds 200 tokens, 192 in the table
    pages = F.pool(g, n, 2, page, 128, "e4m3")
    counts = torch.tensor([20, 7, 99, 4, -1])
    kv = torch.randn(5, Tq, 6, 128, generator=g).to(BF)
    for b in range(5):
        kv[b, :Tq - max(0, min(Tq, int(counts[b])))] = math.nan
    ln = torch.tensor(lengths)
    dev = F.to(pages, "cuda")
    F.append(pages, kv[:, :, 1:3], kv[:, :, 4:6], table, ln, counts)
    on = kv.cuda()
    lsa.append_quantized(dev, on[:, :, 1:3], on[:, :, 4:6], table.cuda(), ln.cuda(), counts.cuda())
    same(dev, pages)


def test_indexes_of_64_bits_that_wrap(lsa):
    """Pages, positions and lengths beyond 32 bits are outside, not what they are modulo 2^32."""
    g = torch.Generator().manual_seed(12)
    pages = lsa.QuantizedPages.new(4, 1, 16, 64)
    k, v = (torch.randn(1, 48, 1, 64, generator=g).cuda() for _ in range(2))
    wrap = 1 << 32
    lsa.append_quantized(pages, k, v, torch.tensor([[1, 2 + wrap, 3]]).cuda(), torch.tensor([48]).cuda())
    assert not bool(pages.k[2].float().any()) and bool(pages.k[3].float().any())
    before = [t.clone() for t in pages]
    lsa.move_pages(pages, torch.tensor([1 + wrap, 1]).cuda(), torch.tensor([0, 2 + wrap]).cuda())
    same(pages, before)
    q = torch.randn(1, 1, 2, 64, generator=g).to(BF).cuda()
    hole = torch.tensor([[1, -1, 3]], dtype=torch.int32).cuda()
    want = lsa.quantized_attention(q, pages, hole, torch.tensor([48]).cuda())
    for table, length in (([1, 2 + wrap, 3], 48), ([1, -1, 3], wrap + 5)):
        # of the second, more tokens than the table has room for: all of its keys
        assert torch.equal(lsa.quantized_attention(q, pages, torch.tensor([table]).cuda(), torch.tensor([length]).cuda()), want)
    lists = torch.tensor([[0, 3 + wrap, 40, -wrap]]).cuda()
    one = lsa.quantized_read(q, pages, hole, torch.tensor([48]).cuda(), lists, torch.tensor([wrap + 3]).cuda())
    two = lsa.quantized_read(q, pages, hole, torch.tensor([48]).cuda(), torch.tensor([[0, 40]]).cuda(),
                             torch.tensor([2]).cuda(), torch.tensor([0]).cuda())
    assert torch.equal(one, two)


def test_append_and_move_of_nothing(lsa):
    pages = lsa.QuantizedPages.new(2, 1, 16, 64)
    before = [t.clone() for t in pages]
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    lsa.append_quantized(pages, torch.ones(0, 1, 1, 64, device="cuda"), torch.ones(0, 1, 1, 64, device="cuda"),
                         none.view(0, 1), none)
    lsa.append_quantized(pages, torch.ones(1, 0, 1, 64, device="cuda"), torch.ones(1, 0, 1, 64, device="cuda"),
                         torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda"))
    lsa.move_pages(pages, none, none)
    same(pages, before)


@pytest.mark.parametrize("code,Hkv,page,D,n", [("e4m3", 8, 64, 128, 40), ("int8", 1, 16, 64, 3), ("e4m3", 3, 128, 128, 11)])
def test_move(lsa, code, Hkv, page, D, n):
    g = torch.Generator().manual_seed(14)
    pages = F.pool(g, 2 * n + 4, Hkv, page, D, code)
    ids = torch.randperm(2 * n + 4, generator=g)
    src, dst = ids[:n + 2].clone(), ids[n + 2:].clone()
    src[0], dst[1] = -1, 2 * n + 4  # skipped
    dev = F.to(pages, "cuda")
    F.move(pages, src, dst)
    lsa.move_pages(dev, src.cuda(), dst.to(torch.int32).cuda())
    same(dev, pages)


# ------------------------------------------------------------------ streams, graphs, the cache


def test_on_another_stream_and_captured(lsa):
    """A step (append, attention) on a stream of its own, captured twice, replayed in turn, equals the eager ones."""
    g = torch.Generator().manual_seed(15)
    cases = []
    for lengths, Tq in (([3000, 65], 1), ([300, 90], 40)):
        table, n = F.paged(g, lengths, 64)
        pages = F.to(F.pool(g, n, 2, 64, 128, "e4m3"), "cuda")
        q = torch.randn(2, Tq, 8, 128, generator=g).to(BF).cuda()
        k, v = (torch.randn(2, Tq, 2, 128, generator=g).to(BF).cuda() for _ in range(2))
        cases.append((pages, q, k, v, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()))

    def step(c):
        pages, q, k, v, table, ln = c
        lsa.append_quantized(pages, k, v, table, ln)
        return lsa.quantized_attention(q, pages, table, ln)

    want = [step(c) for c in cases]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = [step(c) for c in cases]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    graphs, outs = [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(c))
        graphs.append(graph)
    for _ in range(3):
        for o in outs:
            o.zero_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, outs))


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_cache_serves_forks_and_frees(lsa, code):
    """Prompts, ragged ones among them, decode steps, forks that write, places freed and taken again, a compaction:
    every output against the cache's own pages in 64 bits, and the pages against a cache without forks."""
    g = torch.Generator().manual_seed(16)
    Hkv, Hq, D, page = 2, 8, 128, 16
    cache = lsa.QuantizedCache(6, 40, Hkv, D, page, F.CODES[code])
    told = {}  # what every place was given, in order

    def rnd(*shape):
        return torch.randn(*shape, generator=g).to(BF)

    def check(places, q):
        table, ln, _ = cache._upload(places)
        want, _, off, _ = F.attention(q, F.to(cache.pages, "cpu"), table.cpu(), ln.cpu())
        return want, off

    def give(places, Tq, counts=None):
        k, v = rnd(len(places), Tq, Hkv, D), rnd(len(places), Tq, Hkv, D)
        for i, p in enumerate(places):
            c = Tq if counts is None else counts[i]
            if c:
                told.setdefault(p, []).append((k[i:i + 1, Tq - c:], v[i:i + 1, Tq - c:]))
        return k.cuda(), v.cuda()

    cache.append([0, 1], *give([0, 1], 50))
    cache.append([2, 3], *give([2, 3], 30, [30, 7]), counts=[30, 7])
    child = cache.fork(0)
    told[child] = list(told[0])
    assert child == 4 and cache.free_pages == 40 - 4 - 4 - 2 - 1
    for _ in range(20):
        places = [0, child, 3]
        q = rnd(3, 1, Hq, D)
        k, v = give(places, 1)
        out = cache.step(places, q.cuda(), k, v)
        want, off = check(places, q)
        close(out, want, off)
    cache.free([1])
    told.pop(1)
    grand = cache.fork(child)
    assert grand == 1
    told[grand] = list(told[child])
    cache.append([grand, 0], *give([grand, 0], 5))
    held = {p: list(x) for p, x in enumerate(cache._held)}
    used = cache.compact()
    assert used == 40 - cache.free_pages == len({p for x in cache._held for p in x})
    assert max(p for x in cache._held for p in x) == used - 1 and held != {p: list(x) for p, x in enumerate(cache._held)}
    q = rnd(4, 3, Hq, D)
    places = [grand, 3, 0, child]
    k, v = give(places, 3)
    out = cache.step(places, q.cuda(), k, v)
    want, off = check(places, q)
    close(out, want, off)
    lists = torch.randint(0, 30, (2, 9), generator=g, dtype=torch.int32)
    counts = torch.tensor([9, 4], dtype=torch.int32)
    q = rnd(2, 1, Hq, D)
    table, ln, _ = cache._upload([0, 2])
    want, off = F.read(q, F.to(cache.pages, "cpu"), table.cpu(), ln.cpu(), lists, counts, torch.arange(2))
    close(cache.read([0, 2], q.cuda(), lists.cuda(), counts.cuda()), want, off)
    # the same tokens given in the same steps to places that share nothing
    for p, steps in told.items():
        alone = lsa.QuantizedCache(1, 16, Hkv, D, page, F.CODES[code])
        for k, v in steps:
            alone.append([0], k.cuda(), v.cuda())
        assert alone.lengths[0] == cache.lengths[p]
        ids = torch.arange(cache.lengths[p])
        a = F.keys(F.to(alone.pages, "cpu"), alone._upload([0])[0][0].cpu(), ids)
        b = F.keys(F.to(cache.pages, "cpu"), cache._upload([p])[0][0].cpu(), ids)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_step_of_the_whole_path(lsa):
    """Norms and rotation, append, attention, as a model's layer calls them, against the three definitions in a row."""
    from test_gpu_rotate import plain

    g = torch.Generator().manual_seed(17)
    B, T, Hq, Hkv, D = 2, 37, 8, 2, 128
    f, amplitude = lsa.rotary_frequencies(D, 500000.0, "yarn", 4.0, 8192)
    qkv = torch.randn(B, T, Hq + 2 * Hkv, D, generator=g).to(BF).cuda()
    qw, kw = (torch.rand(D, generator=g) + 0.5 for _ in range(2))
    pos = torch.arange(T)
    q, k = lsa.norm_rotate(qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv], pos.cuda(), f.cuda(), qw.cuda(), kw.cuda(),
                           amplitude=amplitude)
    for got, x, w in ((q, qkv[:, :, :Hq], qw), (k, qkv[:, :, Hq:Hq + Hkv], kw)):
        want, off = plain(x.cpu(), pos.expand(B, T), f, w, 1e-6, False, amplitude)
        close(got, want, off)
    cache = lsa.QuantizedCache(2, 8, Hkv, D, 16)
    cache.append([0, 1], k[:, :30], qkv[:, :30, Hq + Hkv:])
    out = cache.step([0, 1], q[:, 30:], k[:, 30:], qkv[:, 30:, Hq + Hkv:])
    table, ln, _ = cache._upload([0, 1])
    pages = lsa.QuantizedPages.new(8, Hkv, 16, D, device="cpu")
    F.append(pages, k[:, :30].cpu(), qkv[:, :30, Hq + Hkv:].cpu(), table.cpu(), torch.tensor([30, 30]))
    F.append(pages, k[:, 30:].cpu(), qkv[:, 30:, Hq + Hkv:].cpu(), table.cpu(), torch.tensor([T, T]))
    want, _, off, _ = F.attention(q[:, 30:].cpu(), pages, table.cpu(), ln.cpu())
    close(out, want, off)


@pytest.mark.parametrize("code,dtype,D,page,group,Hkv,R,W", [
    ("e4m3", BF, 128, 64, 128, 1, 8, 2116), ("int8", HF, 64, 16, 64, 1, 32, 2116), ("e4m3", HF, 64, 32, 33, 2, 40, 1100),
    ("int8", BF, 128, 128, 71, 1, 64, 1030), ("e4m3", BF, 64, 64, 129, 1, 6, 3000)])
def test_read_of_wide_groups(lsa, code, dtype, D, page, group, Hkv, R, W):
    """Groups of more heads than a row tile, on so many keys that rows of a dense call would be the tensor cores': the
    lists count, and the table rows they name - repeated, fewer than the query rows, some outside the table."""
    g = torch.Generator().manual_seed(group)
    lengths = [4000, 0, 33, 2900, 517]
    table, n = F.paged(g, lengths, page)
    table[3, 1] = -1
    pages = F.pool(g, n, Hkv, page, D, code)
    F.poison(pages, table, lengths)
    rows = torch.tensor([0, 3, 0, 4, 1, 9, -1, 2, 3, 0], dtype=torch.int32).repeat(-(-R // 10))[:R]
    lists = torch.stack([torch.randperm(4100, generator=g)[:W] for _ in range(R)]).to(torch.int32)
    counts = torch.randint(0, W + 1, (R,), generator=g, dtype=torch.int32)
    counts[0], counts[1], counts[2] = W, W, 0
    q = torch.randn(R, 1, group * Hkv, D, generator=g).to(dtype)
    ln = torch.tensor(lengths, dtype=torch.int32)
    want, off = F.read(q, pages, table, ln, lists, counts, rows)
    assert bool((want[1] != 0).all())
    got = lsa.quantized_read(q.cuda(), F.to(pages, "cuda"), table.cuda(), ln.cuda(), lists.cuda(), counts.cuda(), rows.cuda())
    close(got, want, off)
    assert bool((got[[2, 4, 5]] == 0).all())


def test_append_of_no_token_leaves_the_page(lsa):
    """A count of 0 (or a negative one) on a partly full page writes nothing, whatever scale the caller gave the page;
    its neighbour in the call is written."""
    g = torch.Generator().manual_seed(24)
    for Tq in (1, 3, 20):  # a warp a page, a CTA a page
        for code in ("e4m3", "int8"):
            pages = F.pool(g, 5, 2, 32, 64, code)
            for s in (pages.k_scale, pages.v_scale):
                s.copy_(torch.tensor([2.0 ** -70, 0.75 * 2.0 ** -63, 2.0 ** -70, 1.0, 2.0 ** -70])[:, None].expand(5, 2))
            table = torch.tensor([[0, -1], [1, 4], [2, 3]], dtype=torch.int32)
            ln, counts = torch.tensor([20, 40, 25]), torch.tensor([0, 1, -3])
            dev = F.to(pages, "cuda")
            k, v = (torch.randn(3, Tq, 2, 64, generator=g) for _ in range(2))
            F.append(pages, k, v, table, ln, counts)
            lsa.append_quantized(dev, k.cuda(), v.cuda(), table.cuda(), ln.cuda(), counts.cuda())
            same(dev, pages)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dtype,D,page,code", [(BF, 128, 64, "e4m3"), (HF, 64, 16, "int8"), (HF, 128, 32, "e4m3")])
@pytest.mark.parametrize("Tq,Hq,Hkv", [(1, 4, 1), (3, 4, 1), (5, 16, 4), (40, 32, 8), (70, 32, 8)],
                         ids=["8rows", "16rows", "32rows", "two halves", "many rows"])
def test_rows_without_keys_read_as_zeros_whatever_they_hold(lsa, Tq, Hq, Hkv, dtype, D, page, code, bad):
    """Rows of q that are not finite and see no key - all pages that they see unmapped, or before token 0 - are zeros
    with log-sum-exp -inf; the rows beside them, of the same tile, are as they were."""
    g = torch.Generator().manual_seed(25)
    lengths = [Tq // 2, 700, page + Tq - 1, 0, 1150, 130, 900, 1000, 300, 40]
    table, n = F.paged(g, lengths, page)
    table[1] = -1
    table[2, :1] = 1 << 30  # its first row sees this page only
    table[4, ::2] = -1
    pages = F.pool(g, n, Hkv, page, D, code)
    F.poison(pages, table, lengths)
    q = torch.randn(len(lengths), Tq, Hq, D, generator=g).to(dtype)
    ln = torch.tensor(lengths, dtype=torch.int32)
    want, want_lse, off, lse_off = F.attention(q, pages, table, ln)
    none = want_lse == -math.inf
    assert bool(none[1].all()) and bool(none[2, 0].all()) and not bool(none[4].any())
    q[none] = bad
    got, lse = lsa.quantized_attention(q.cuda(), F.to(pages, "cuda"), table.cuda(), ln.cuda(), return_lse=True)
    assert bool((got[none.cuda()] == 0).all()) and bool((lse[none.cuda()] == -math.inf).all())
    close(got, want, off)
    close(lse, want_lse, lse_off + 2.0 ** -22)


@pytest.mark.parametrize("dtype,group", [(BF, 4), (HF, 16), (BF, 40)])
def test_reads_without_keys_are_zeros_whatever_they_hold(lsa, dtype, group):
    g = torch.Generator().manual_seed(26)
    lengths = [300, 0, 300, 300]
    table, n = F.paged(g, lengths, 32)
    table[2] = -1
    pages = F.pool(g, n, 2, 32, 64, "e4m3")
    q = torch.randn(5, 1, 2 * group, 64, generator=g).to(dtype)
    lists = torch.randint(0, 300, (5, 200), generator=g, dtype=torch.int32)
    lists[3] = 300
    counts, rows = torch.tensor([0, 200, 200, 200, 200]), torch.tensor([0, 1, 2, 3, 0])
    ln = torch.tensor(lengths)
    want, off = F.read(q, pages, table, ln, lists, counts, rows)
    q[:4] = torch.tensor([math.nan, math.inf, -math.inf, math.nan]).view(4, 1, 1, 1).to(dtype)
    got = lsa.quantized_read(q.cuda(), F.to(pages, "cuda"), table.cuda(), ln.cuda(), lists.cuda(), counts.cuda(), rows.cuda())
    assert bool((got[:4] == 0).all())
    close(got, want, off)


def test_cache_calls_do_not_wait_for_the_device(lsa, monkeypatch):
    """Appends, steps, attention, reads and a fork's copies return while the stream is still busy with what came before
    them (the checked mode waits by itself), and what they uploaded is what their kernels find."""
    monkeypatch.delenv("LSA_CHECK_STATUS", raising=False)
    g = torch.Generator().manual_seed(27)
    Hkv, Hq, D = 2, 8, 64
    k, v = (torch.randn(2, 40, Hkv, D, generator=g).to(BF).cuda() for _ in range(2))
    q = torch.randn(2, 2, Hq, D, generator=g).to(BF).cuda()
    lists, counts = torch.randint(0, 40, (2, 9), generator=g).cuda(), torch.tensor([9, 5]).cuda()

    def use(busy):
        cache = lsa.QuantizedCache(4, 64, Hkv, D, 16)
        torch.cuda.synchronize()
        done = torch.cuda.Event()
        if busy:
            torch.cuda._sleep(1 << 29)  # a quarter of a second
            done.record()
        outs, early = [], []
        for call in (lambda: cache.append([0, 1], k, v), lambda: cache.step([0, 1], q, k[:, :2], v[:, :2]),
                     lambda: cache.step([cache.fork(0), 0], q, k[:, 2:4], v[:, 2:4]), lambda: cache.attend([1, 0], q),
                     lambda: cache.free([1]), cache.compact, lambda: cache.read([2, 0], q[:, :1], lists, counts)):
            out = call()
            early.append(busy and not done.query())
            outs.append(out)
        torch.cuda.synchronize()
        return [x for x in outs if torch.is_tensor(x)], early

    want, _ = use(False)
    use(True)  # buffers of this many calls in flight at once
    got, early = use(True)
    assert all(early), early
    assert len(want) == 4 and all(torch.equal(a, b) for a, b in zip(want, got))


def weights_case(g, lengths, Tq, Hkv, group, D, page, code):
    """Values of alternating sign with nearly equal weights, which all but cancel: what their rounding costs is not hidden
    by the output's own."""
    table, n = F.paged(g, lengths, page)
    pages = F.pool(g, n, Hkv, page, D, code)
    sign = (1 - 2 * (torch.arange(page) & 1))[None, None, :, None] * (1 - 2 * torch.randint(0, 2, (n, Hkv, 1, D), generator=g))
    pages.v.copy_(sign.float().to(pages.v.dtype))
    pages.v_scale.fill_(1.0)
    F.poison(pages, table, lengths)
    return pages, table, torch.tensor(lengths, dtype=torch.int32), torch.randn(len(lengths), Tq, Hkv * group, D, generator=g)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("B,Tq,Hkv,group,D,page,code", [(40, 1, 2, 4, 128, 64, "e4m3"), (40, 3, 2, 4, 64, 16, "int8"),
                                                        (40, 5, 1, 6, 128, 32, "e4m3"), (16, 40, 8, 4, 128, 64, "e4m3"),
                                                        (16, 70, 8, 4, 64, 16, "int8")])
def test_weights_are_rounded_to_11_bits(lsa, B, Tq, Hkv, group, D, page, code, dtype):
    """Off by 2^-11 of each weight at most, besides the output's rounding - also where q and the output are bf16. Weights
    of 8 bits, as a bf16's, would not pass."""
    g = torch.Generator().manual_seed(28)
    lengths = [Tq + 1 + i % 5 for i in range(B)]
    pages, table, ln, q = weights_case(g, lengths, Tq, Hkv, group, D, page, code)
    q, scale = q.to(dtype), 0.05 * D ** -0.5
    want = torch.zeros(q.shape, dtype=torch.float64)
    off, worse = torch.zeros_like(want), torch.zeros_like(want)
    for b, n in enumerate(lengths):
        ids, key, val = F.keys(pages, table[b], torch.arange(n))
        seen = ids[None, :] < (n - Tq + torch.arange(Tq) + 1)[:, None]
        for h in range(q.shape[2]):
            x, k, v = q[b, :, h].double(), key[:, h // group], val[:, h // group]
            out, _, o, _ = F.rows(x, k, v, scale, seen, 2.0 ** -11)
            logits = (x @ k.T * scale).masked_fill(~seen, -math.inf)
            p = torch.exp(logits - logits.amax(-1, keepdim=True))
            want[b, :, h], off[b, :, h] = out, o
            worse[b, :, h] = p.to(BF).double() @ v / p.sum(-1, keepdim=True)
    off += torch.finfo(dtype).eps / 2 * want.abs()
    assert ((worse - want).abs() > off).double().mean() > 0.01
    got = lsa.quantized_attention(q.cuda(), F.to(pages, "cuda"), table.cuda(), ln.cuda(), scale)
    close(got, want, off)
    if Tq == 1:
        lists = torch.arange(8, dtype=torch.int32).expand(B, 8).contiguous()
        close(lsa.quantized_read(q.cuda(), F.to(pages, "cuda"), table.cuda(), ln.cuda(), lists.cuda(), ln.cuda(), scale=scale),
              want, off)


def test_cache_calls_of_no_place_and_under_a_default_device(lsa):
    g = torch.Generator().manual_seed(29)
    cache = lsa.QuantizedCache(3, 8, 2, 64, 16)
    none = torch.empty(0, 3, 2, 64, device="cuda", dtype=BF)
    cache.append([], none, none)
    assert cache.step([], none, none, none).shape == none.shape and cache.attend([], none).shape == none.shape
    k, v, q = (torch.randn(2, 9, 2, 64, generator=g).to(BF).cuda() for _ in range(3))
    lists, counts = torch.randint(0, 9, (2, 5), generator=g).cuda(), torch.tensor([5, 2]).cuda()

    def use():
        cache.append([0, 1], k, v)
        out = cache.step([1, cache.fork(0)], q[:, :2], k[:, :2], v[:, :2])
        out2 = cache.read([0, 1], q[:, :1], lists, counts)
        cache.free([0])
        cache.compact()
        out3 = cache.attend([2, 1], q)
        cache.free([0, 1, 2])
        return out, out2, out3

    want = use()
    with torch.device("cuda"):
        got = use()
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and cache.free_pages == 8


@pytest.mark.parametrize("group,Hkv,R,W", [(4, 2, 12, 700), (64, 1, 32, 2116), (128, 1, 8, 2116)])
def test_reads_captured_and_on_another_stream(lsa, group, Hkv, R, W):
    """Two reads captured in graphs of their own, replayed in turn and beside an eager one on another stream."""
    g = torch.Generator().manual_seed(30)
    lengths = [4000, 2500, 900]
    table, n = F.paged(g, lengths, 64)
    pages = F.to(F.pool(g, n, Hkv, 64, 128, "e4m3"), "cuda")
    table, ln = table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()
    args = []
    for _ in range(2):
        q = torch.randn(R, 1, group * Hkv, 128, generator=g).to(BF)
        q[1] = math.nan
        lists, counts = torch.randint(0, 4000, (R, W), generator=g, dtype=torch.int32), torch.randint(1, W + 1, (R,), generator=g)
        counts[1] = 0
        args.append((q.cuda(), lists.cuda(), counts.to(torch.int32).cuda(), torch.randint(0, 3, (R,), generator=g).to(torch.int32).cuda()))

    def read(a):
        return lsa.quantized_read(a[0], pages, table, ln, *a[1:])

    want = [read(a) for a in args]
    assert all(bool((w[1] == 0).all()) and bool(w.isfinite().all()) for w in want)
    graphs, outs = [], []
    for a in args:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(read(a))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        for o, graph in zip(outs, graphs):
            o.zero_()
            graph.replay()
        with torch.cuda.stream(side):
            beside = read(args[0])
        torch.cuda.synchronize()
        assert torch.equal(beside, want[0]) and all(torch.equal(a, b) for a, b in zip(outs, want))
