"""The 8-bit paged cache on the host: refusals, the cache's books, the frequencies, the tests' own definitions."""

import math

import pytest
import torch

import quantized_forms as F


@pytest.fixture()
def plain(monkeypatch, lsa):
    """The cache's operators from their definitions, on CPU tensors."""
    from lsa_b200 import quantized

    monkeypatch.setattr(quantized, "append_quantized", F.append)
    monkeypatch.setattr(quantized, "move_pages", F.move)
    monkeypatch.setattr(quantized, "quantized_attention",
                        lambda q, pages, table, ln, scale=None: F.attention(q, pages, table, ln, scale)[0].to(q.dtype))
    return quantized


def given(n, T, seed=0, Hkv=1, D=64):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, T, Hkv, D, generator=g), torch.randn(n, T, Hkv, D, generator=g)


def books(cache):
    """References and free pages agree with what the places hold."""
    held = [p for x in cache._held for p in x]
    assert [held.count(p) for p in range(len(cache._refs))] == cache._refs
    assert sorted(cache._free) == [p for p, r in enumerate(cache._refs) if r == 0]
    assert all(len(x) == -(-n // cache.page) for x, n in zip(cache._held, cache.lengths))


def test_cache_books(plain):
    cache = plain.QuantizedCache(4, 8, 1, 64, 16, device="cpu")
    cache.append([0], *given(1, 20))
    child = cache.fork(0)
    books(cache)
    assert child == 1 and cache.free_pages == 6
    before = [t.clone() for t in cache.pages]
    cache.append([child], *given(1, 3, 1))  # the shared, partly full page is copied, the full one is not
    books(cache)
    assert cache._held[0][0] == cache._held[1][0] and cache._held[0][1] != cache._held[1][1]
    p = cache._held[0][1]
    assert all(torch.equal(a[p].float(), b[p].float()) for a, b in zip(before, cache.pages))
    cache.append([0], *given(1, 3, 2))  # alone on its page now: no copy
    books(cache)
    assert cache._held[0][1] == p and cache.free_pages == 5
    cache.free([0])
    books(cache)
    assert cache.lengths[0] == 0 and cache.free_pages == 6
    cache.append([2], *given(1, 60, 3))
    cache.free([child])
    keys = F.keys(cache.pages, torch.tensor(cache._held[2]), torch.arange(60))
    assert cache.compact() == 4 and cache._held[2] and max(cache._held[2]) == 3
    books(cache)
    after = F.keys(cache.pages, torch.tensor(cache._held[2]), torch.arange(60))
    assert all(torch.equal(a, b) for a, b in zip(keys, after))


def test_both_of_a_fork_write_in_one_call(plain):
    cache = plain.QuantizedCache(3, 6, 1, 64, 16, device="cpu")
    cache.append([0], *given(1, 5))
    a, b = cache.fork(0), cache.fork(0)
    cache.append([0, a, b], *given(3, 2, 1))
    books(cache)
    assert len({x[0] for x in cache._held}) == 3 and cache.free_pages == 3


def test_an_empty_place_has_no_fork(plain):
    cache = plain.QuantizedCache(3, 6, 1, 64, 16, device="cpu")
    with pytest.raises(ValueError):
        cache.fork(0)  # its fork would be place 1, and the next fork's too
    cache.append([0], *given(1, 5))
    assert cache.fork(0) == 1 and cache.fork(0) == 2


def test_cache_refusals_leave_it_as_it_was(plain):
    cache = plain.QuantizedCache(2, 3, 2, 64, 16, device="cpu")
    k, v = given(1, 30, Hkv=2)
    cache.append([0], k, v)
    state = (list(cache.lengths), [list(x) for x in cache._held], list(cache._refs), list(cache._free),
             [t.clone() for t in cache.pages])

    def refused(fn, *args, **kw):
        with pytest.raises(ValueError):
            fn(*args, **kw)
        assert state[:4] == (list(cache.lengths), [list(x) for x in cache._held], list(cache._refs), list(cache._free))
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(state[4], cache.pages))

    q = torch.randn(1, 30, 4, 64).to(torch.bfloat16)
    refused(cache.append, [0], *given(1, 19, Hkv=2))  # two pages more, one free
    refused(cache.append, [0, 0], *given(2, 1, Hkv=2))
    refused(cache.append, [2], k, v)
    refused(cache.append, [-1], k, v)
    refused(cache.append, [0, 1], k, v)
    refused(cache.append, [0], k[..., :1, :], v[..., :1, :])
    refused(cache.append, [0], k, v[:, :29])
    refused(cache.append, [0], k.double(), v.double())
    refused(cache.append, [0], k, v, counts=[31])
    refused(cache.append, [0], k, v, counts=[1, 1])
    refused(cache.step, [0], q[:, :3], k[:, :2], v[:, :2])
    refused(cache.step, [0], q[:, :2].float(), k[:, :2], v[:, :2])
    refused(cache.step, [0], q[:, :2, :3], k[:, :2], v[:, :2])
    refused(cache.step, [0], q[:, :2], k[:, :2], v[:, :2], scale=0.0)
    # rows that the attention has no grid for, before anything is appended
    refused(cache.step, [0], q[:1, :1, :1].expand(1, 1 << 24, 128, 64), k[:1, :1].expand(1, 1 << 24, 2, 64),
            v[:1, :1].expand(1, 1 << 24, 2, 64))
    refused(cache.attend, [0, 1], q)
    refused(cache.fork, 5)
    cache.append([1], *given(1, 3, Hkv=2))
    with pytest.raises(ValueError):
        cache.fork(0)  # no free place


@pytest.mark.parametrize("bad", [dict(places=0), dict(places=65536), dict(pages=0), dict(page=24), dict(head_dim=96), dict(kv_heads=0),
                                 dict(dtype=torch.uint8)])
def test_cache_sizes_refused(lsa, bad):
    with pytest.raises(ValueError):
        lsa.QuantizedCache(**{**dict(places=1, pages=1, kv_heads=1, head_dim=64, device="cpu"), **bad})


def test_cpu_tensors_are_refused(lsa):
    pages = lsa.QuantizedPages.new(2, 1, 16, 64, device="cpu")
    q = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    k = torch.zeros(1, 1, 1, 64)
    table, ln = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    f, _ = lsa.rotary_frequencies(64)
    for call in (lambda: lsa.quantized_attention(q, pages, table, ln), lambda: lsa.append_quantized(pages, k, k, table, ln),
                 lambda: lsa.quantized_read(q, pages, table, ln, table, ln), lambda: lsa.move_pages(pages, ln, ln),
                 lambda: lsa.norm_rotate(k, k, torch.zeros(1, 1, dtype=torch.int32), f)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_shapes_without_a_device(lsa):
    """The operators' Meta forms."""
    from lsa_b200 import _lib

    ops = _lib.torch_ops()
    q, k = torch.empty(2, 3, 8, 128, device="meta", dtype=torch.bfloat16), torch.empty(2, 3, 2, 128, device="meta")
    pool = [torch.empty(5, 2, 16, 128, device="meta", dtype=torch.int8)] * 2 + [torch.empty(5, 2, device="meta")] * 2
    table, ln = torch.empty(2, 4, device="meta", dtype=torch.int32), torch.empty(2, device="meta", dtype=torch.int32)
    out, lse = ops.quantized_attention_lse(q, *pool, table, ln, 0.1)
    assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (2, 3, 8) and lse.dtype == torch.float32
    assert ops.quantized_attention(q, *pool, table, ln, 0.1).shape == q.shape
    assert ops.quantized_read(q[:, :1], *pool, table, ln, table, ln, None, 0.1).shape == (2, 1, 8, 128)
    a, b = ops.norm_rotate(q, q[:, :, :2], ln, ln, None, None, 1e-6, False, 1.0)
    assert a.shape == q.shape and b.shape == (2, 3, 2, 128)
    ops.append_quantized(k, k, *pool, table, ln)
    ops.move_pages(*pool, ln, ln)


def test_entry_points_refuse_before_any_launch(lsa):
    """The C entries' status for arguments that they do not take (no device is touched)."""
    from lsa_b200 import _lib
    from lsa_b200._lib import ERR_ARG, ERR_SIZE, OK

    L = _lib.lib()
    import ctypes

    some = ctypes.c_void_p(4096)
    st = (ctypes.c_int64 * 6)(*[128] * 6)
    odd = (ctypes.c_int64 * 6)(128, 128, 129, 128, 128, 128)

    def rotate(dtype=2, s=st, B=1, T=1, Hq=2, Hkv=1, D=128, R=64, qp=some, wd=0):
        return L.lsa_norm_rotate(qp, some, dtype, s, B, T, Hq, Hkv, D, some, 0, 0, 1, some, R, 0, 1.0, some, wd, None, 0,
                                 1e-6, some, some, None)

    for bad in (dict(dtype=3), dict(s=odd), dict(Hq=0), dict(D=96), dict(R=24), dict(R=144), dict(wd=1), dict(B=-1),
                dict(qp=ctypes.c_void_p(4100)), dict(qp=None)):
        assert rotate(**bad) == ERR_ARG, bad
    assert rotate(B=0) == OK

    def append(dtype=2, code=0, pages=4, page=16, M=1, B=1, Tq=1, Hkv=1, D=64, s=st, k=some):
        return L.lsa_append_quantized(k, some, dtype, s, some, some, some, some, code, pages, page, some, 1, M, some, None,
                                      B, Tq, Hkv, D, None)

    for bad in (dict(dtype=5), dict(code=2), dict(page=24), dict(D=96), dict(s=odd), dict(k=None), dict(Tq=-1)):
        assert append(**bad) == ERR_ARG, bad
    assert append(Tq=0) == OK and append(M=0) == OK and append(B=0) == OK

    def attend(dtype=2, code=0, pages=4, page=16, M=1, B=1, Tq=1, Hq=2, Hkv=1, D=64, scale=0.1, bytes_=1 << 40, s=st,
               status=some):
        return L.lsa_quantized_attention(some, dtype, s, some, some, some, some, code, pages, page, some, 1, M, some, B, Tq,
                                         Hq, Hkv, D, scale, some, None, some, bytes_, status, None)

    for bad in (dict(dtype=0), dict(code=-1), dict(page=48), dict(Hq=3, Hkv=2), dict(D=256), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(M=1 << 40), dict(s=odd),
                dict(status=None), dict(M=4096, bytes_=0)):
        assert attend(**bad) == ERR_ARG, bad
    assert attend(pages=1 << 28) == ERR_SIZE
    assert attend(B=0) == OK and attend(Tq=0) == OK

    def read(R=1, W=4, table_rows=1, rows=None, counts=some):
        return L.lsa_quantized_read(some, 2, st, some, some, some, some, 0, 4, 16, some, 1, table_rows, 1, some, some, counts,
                                    rows, R, W, 2, 1, 64, 0.1, some, None, 0, None)

    assert read(R=2) == ERR_ARG and read(counts=None) == ERR_ARG and read(W=-1) == ERR_ARG and read(R=0) == OK
    assert L.lsa_move_pages(some, some, some, some, 4, 24, 1, 64, some, some, 1, None) == ERR_ARG
    assert L.lsa_move_pages(some, some, some, some, 4, 16, 1, 64, some, some, 0, None) == OK
    # query heads beyond the tensor cores' tiles: rows without a grid
    assert L.lsa_quantized_scratch(1, 1 << 13, 256, 1, 64, 4096, 0) == ERR_SIZE
    assert L.lsa_quantized_scratch(1, 1 << 12, 256, 1, 64, 4096, 0) >= 0
    assert all(L.lsa_quantized_scratch(1, 1 << 20, 16, 4, 64, n, 0) >= 0 for n in (0, 16, 64, 4096))
    assert L.lsa_quantized_scratch(1, 1, 3, 2, 64, 100, 0) == ERR_ARG and L.lsa_quantized_scratch(0, 1, 2, 1, 64, 100, 0) == 0


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_nearest_agrees_with_torch(code):
    g = torch.Generator().manual_seed(0)
    x = torch.cat([torch.randn(20000, generator=g) * 3, torch.arange(-448, 449) / 2.0, torch.arange(-64, 65) * 2.0 ** -11])
    x = x.clamp(-F.QMAX[code], F.QMAX[code])
    want = x.to(torch.float8_e4m3fn).double() if code == "e4m3" else x.round().double()
    assert torch.equal(F.nearest(x.double(), code), want)


def test_frequencies(lsa):
    f, a = lsa.rotary_frequencies(64, 10000.0)
    assert a == 1.0 and f.dtype == torch.float64 and f.numel() == 32
    assert abs(float(f[5]) - 10000.0 ** (-10 / 64)) < 1e-15
    g, a = lsa.rotary_frequencies(64, 10000.0, "linear", 4.0)
    assert a == 1.0 and torch.equal(g, f / 4)
    g, a = lsa.rotary_frequencies(64, 10000.0, "ntk", 4.0)
    assert float(g[0]) == 1.0 and abs(float(g[-1]) / float(f[-1]) - 0.25) < 1e-12  # the slowest pair by the factor
    g, a = lsa.rotary_frequencies(64, 10000.0, "yarn", 8.0, 4096)
    turns = f * 4096 / (2 * math.pi)
    assert torch.allclose(g[turns > 40], f[turns > 40]) and torch.allclose(g[turns < 0.8], f[turns < 0.8] / 8)
    assert bool((g <= f).all()) and bool((g >= f / 8).all()) and abs(a - (0.1 * math.log(8) + 1)) < 1e-15
    for bad in ((63,), (0,), (64, 1.0), (64, 1e4, "other"), (64, 1e4, "linear", 0.5), (64, 1e4, "yarn", 2.0),
                (64, math.inf), (64, 1e4, "yarn", 2.0, 4096, 1.0, 2.0)):
        with pytest.raises(ValueError):
            lsa.rotary_frequencies(*bad)


@pytest.mark.parametrize("Hkv", [1, 2])
@pytest.mark.parametrize("group", [31, 33, 47, 71, 127, 129])
@pytest.mark.parametrize("R,W", [(1, 16385), (8, 2116), (64, 2116), (700, 300)])
def test_reads_are_planned_by_their_own_rows(lsa, R, W, group, Hkv):
    """A read's scratch is whole parts of its R rows a head, whatever the group: the kernel that knows lists plans it. (The
    tensor cores' tiles of 128 rows, which the odd groups do not divide, hold no lists.)"""
    from lsa_b200 import _lib

    one = R * group * Hkv * (128 + 1) * 4
    got = _lib.lib().lsa_quantized_scratch(R, 1, group * Hkv, Hkv, 128, W, 1)
    assert got >= 0 and got % one == 0 and got // one <= 96


@pytest.mark.parametrize("scale", [3e38, 1e39, 1e-46, -1e-46, math.nan, math.inf])
def test_a_step_whose_scale_the_operator_refuses_appends_nothing(plain, scale):
    """The operator takes the scale times log2(e) in fp32: 3e38 is an infinity there, 1e-46 a zero."""
    cache = plain.QuantizedCache(1, 4, 2, 64, 16, device="cpu")
    cache.append([0], *given(1, 10, Hkv=2))
    before = [t.clone() for t in cache.pages]
    k, v = given(1, 7, 1, Hkv=2)
    with pytest.raises(ValueError):
        cache.step([0], torch.zeros(1, 7, 4, 64, dtype=torch.bfloat16), k, v, scale=scale)
    assert cache.lengths == [10] and cache.free_pages == 3
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(before, cache.pages))
    for near in (2e38, 1e-38):  # taken by both
        cache.step([0], torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16), k[:, :1], v[:, :1], scale=near)
    assert cache.lengths == [12]


@pytest.mark.parametrize("bad", [dict(kv_heads=65536), dict(kv_heads=1 << 12, pages=1 << 15), dict(pages=(1 << 24) + 1, page=128)])
def test_pools_that_the_operators_refuse_are_no_cache(lsa, bad):
    """Heads beyond a launch's, rows (page, head, token) beyond 2^31 - 1: refused before anything is allocated."""
    with pytest.raises(ValueError):
        lsa.QuantizedCache(**{**dict(places=1, pages=1, kv_heads=1, head_dim=64, page=16, device="meta"), **bad})


@pytest.mark.parametrize("trained,fast,slow", [(4, 32.0, 1.0), (100, 64.0, 32.0), (6, 2.0, 1.0), (4096, 32.0, 1.0)])
def test_yarn_pairs_below_slow_turns_are_over_the_factor(lsa, trained, fast, slow):
    """The first pair too, where the trained length is too short for it to turn ``slow`` times."""
    f, _ = lsa.rotary_frequencies(64, 10000.0)
    g, _ = lsa.rotary_frequencies(64, 10000.0, "yarn", 8.0, trained, fast, slow)
    below = f * trained / (2 * math.pi) < slow * (1 - 1e-9)
    assert bool(below.any()) and torch.equal(g[below], f[below] / 8)


def test_uploads_are_staged_on_the_host_whatever_the_default_device(plain):
    cache = plain.QuantizedCache(2, 4, 1, 64, 16, device="cpu")
    cache.append([0], *given(1, 20))
    with torch.device("meta"):
        table, lengths, counts = cache._upload([1, 0], [3, 4])
    assert table.tolist() == [[-1, -1], [0, 1]] and lengths.tolist() == [0, 20] and counts.tolist() == [3, 4]
