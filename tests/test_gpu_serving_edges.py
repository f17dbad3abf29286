"""Edges of the shared-prefix attention, the scored attention and the budgeted cache on the GPU."""

import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def test_scores_where_keys_times_heads_pass_32_bits(lsa):
    """64 heads on a cache of just over 2^25 keys: all logits are zero, so every key - the first ones
    among them - gains 64 / n. The weight is a sum of 64 fp32 terms of relative error below 2e-4."""
    n = (1 << 25) + 300
    k = torch.zeros(1, n, 1, 64, dtype=BF, device=DEV)
    q = torch.ones(1, 1, 64, 64, dtype=BF, device=DEV)
    scores = torch.zeros(1, 1, n, device=DEV)
    out, got = lsa.scored_attention(q, k, k, torch.tensor([n], device=DEV), scores)
    assert (out == 0).all()
    assert float((got.double() * n / 64 - 1).abs().max()) <= 2e-4


def light_tail(B, Tq, Hq, Hkv, D, P, T):
    """Every 2048 keys four heavy ones of value zero (16 keys apart), the others 2^-25.3 of their
    weight and all of the output. A key that nothing but the first component tells apart, so a row's
    logits are exact products."""
    g = torch.Generator(device=DEV)
    g.manual_seed(P + T)

    def cache(*shape):
        n = shape[-3]
        j = torch.arange(n, device=DEV)
        heavy = ((j % 16 == 3) & (j // 64 % 32 == 0)).view(*([1] * (len(shape) - 3)), n, 1, 1)
        k = torch.zeros(*shape, device=DEV)
        k[..., 0] = torch.where(heavy[..., 0], 25.3 * math.log(2.0) / 8.0, 0.0)
        v = torch.where(heavy, 0.0, 40.0 + 20.0 * torch.rand(*shape, generator=g, device=DEV))
        return k.to(HF), v.to(HF)

    q = torch.randn(B, Tq, Hq, D, generator=g, device=DEV)
    q[..., 0] = 8.0
    lengths = torch.randint(min(Tq, T), T + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
    return (q.to(HF), *cache(P, Hkv, D), *cache(B, T, Hkv, D), lengths)


@pytest.mark.parametrize("case", [
    (1, 1, 4, 1, 128, 400000, 64),   # few rows, the prefix
    (8, 1, 8, 8, 64, 0, 70000),      # few rows, own caches
    (1, 1, 32, 1, 128, 400000, 64),  # one half's rows, two streams of chunks
    (2, 100, 8, 2, 64, 100000, 500), # row tiles of a sequence that read the prefix, split
    (37, 64, 16, 4, 128, 20000, 64), # the same, whole
    (1, 40, 8, 2, 128, 0, 60000),    # row tiles of a sequence, own keys alone
], ids=lambda c: "-".join(map(str, c)))
def test_light_tails_in_fp16(lsa, case):
    """Weights far below the row's largest keep their mass. fp16 holds a weight to 2^-25 absolute below
    2^-14; the kernels scale the weights by 2^7 or more before they round, so a key is off by at most
    2^-32 of the largest beside the usual bound of the attention's tests (u = 2^-11)."""
    q, kp, vp, k, v, lengths = light_tail(*case)
    B, Tq, Hq, D = q.shape
    P, Hkv, _ = kp.shape
    G, u = Hq // Hkv, 2.0 ** -11
    got = lsa.shared_prefix_attention(q, kp, vp, k, v, lengths, 1.0)
    worst = -math.inf
    for b in range(B):
        n = int(lengths[b])
        for h in range(Hkv):
            key, val = torch.cat([kp[:, h], k[b, :n, h]]).double(), torch.cat([vp[:, h], v[b, :n, h]]).double()
            s = q[b, :, h * G:(h + 1) * G].double().reshape(Tq * G, D) @ key.T
            last = (P + n - Tq + torch.arange(Tq, device=DEV)).repeat_interleave(G)
            s = s.masked_fill(torch.arange(P + n, device=DEV) > last[:, None], -math.inf)
            e = torch.exp(s - s.amax(-1, keepdim=True))
            out = (e @ val) / e.sum(-1, keepdim=True)  # val >= 0: also the sum of p |v|
            lost = 2.0 ** -32 * val.sum(0) / e.sum(-1, keepdim=True)
            x = got[b, :, h * G:(h + 1) * G].double().reshape(Tq * G, D)
            worst = max(worst, float(((x - out).abs() - u * out - (u + 2e-4) * out - lost - 1e-6).max()))
    assert worst <= 0


def budgeted(lsa, B=3, Hkv=2, D=64, dt=BF):
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dt)
    c = lsa.BudgetedCache(r(B, 90, Hkv, D), r(B, 90, Hkv, D), [90, 64, 10], 64, 8, window_size=8, sink_size=2)
    return c, r


def test_a_refused_step_changes_nothing(lsa):
    """New keys of another batch or length (which an indexed write would repeat), of another type, a query
    that the operator refuses: a ValueError, and the cache goes on as if the step had not been tried."""
    cache, r = budgeted(lsa)
    twin, _ = budgeted(lsa)
    B, Hq, Hkv, D = 3, 4, 2, 64
    first = (r(B, 4, Hq, D), r(B, 4, Hkv, D), r(B, 4, Hkv, D))
    assert torch.equal(cache.step(*first), twin.step(*first))
    q, kn, vn = r(B, 5, Hq, D), r(B, 5, Hkv, D), r(B, 5, Hkv, D)  # an eviction is due before it
    bad = [(q, kn[:, :1], vn[:, :1]), (q, kn[:1], vn[:1]), (q, kn[:, :, :1], vn[:, :, :1]), (q, kn, vn[..., :1]),
           (q[:1], kn, vn), (q, kn.float(), vn.float()), (q.half(), kn, vn), (q[:, :, :3], kn, vn), (q[0], kn, vn),
           (q[..., :32], kn, vn), (q, kn.cpu(), vn.cpu()), (q, kn, vn, -1.0), (q, kn, vn, math.nan)]
    for args in bad:
        with pytest.raises(ValueError):
            cache.step(*args)
        assert torch.equal(cache.lengths, twin.lengths) and torch.equal(cache.scores, twin.scores)
    n = int(cache.lengths.max())
    assert torch.equal(cache.k[:, :n], twin.k[:, :n]) and torch.equal(cache.v[:, :n], twin.v[:, :n])
    assert torch.equal(cache.step(q, kn, vn), twin.step(q, kn, vn))
    assert torch.equal(cache.scores, twin.scores) and torch.equal(cache.lengths, twin.lengths)


@pytest.fixture()
def wait_limit():
    """Sets the limit of the tensor-core kernels' waits (ns); the default again afterwards."""
    from lsa_b200 import _lib

    _lib.torch_ops()
    yield lambda ns: _lib.check(_lib.lib().lsa_shared_prefix_wait_limit(ns), "wait limit")
    assert _lib.lib().lsa_shared_prefix_wait_limit(-1) == _lib.OK


@pytest.mark.parametrize("case", [
    (40, 1, 32, 4, 64, 700, 500),   # prefix: two streams of chunks, more tiles than the ring holds
    (40, 5, 32, 4, 128, 200, 200),  # few tiles: all of them in flight at once
    (3, 64, 16, 4, 128, 2000, 300), # both halves, prefix and own keys, split
    (40, 64, 16, 4, 128, 300, 130), # whole tiles
    (2, 32, 32, 8, 128, 0, 3000),   # weights of 128 rows: Q resident
    (1, 257, 6, 2, 64, 0, 400),     # weights of seven row tiles: Q streamed
], ids=lambda c: "-".join(map(str, c)))
def test_expired_waits_leave_with_their_copies_landed(lsa, wait_limit, case):
    """Every role gives up at its first wait, with the first copies in flight. The call reports it, and calls
    after it, on the same SMs, answer as before. (A CTA that left copies behind could have them land in the
    next one's shared memory.)"""
    B, Tq, Hq, Hkv, D, P, T = case
    g = torch.Generator(device=DEV)
    g.manual_seed(T)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(BF)
    q, kp, vp, k, v = r(B, Tq, Hq, D), r(P, Hkv, D), r(P, Hkv, D), r(B, T, Hkv, D), r(B, T, Hkv, D)
    lengths = torch.randint(min(Tq, T), T + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
    scores = torch.rand(B, Hkv, T, generator=g, device=DEV)
    call = lambda: lsa.scored_attention(q, k, v, lengths, scores, k_prefix=kp, v_prefix=vp)
    want = call()
    for _ in range(3):
        wait_limit(0)
        with pytest.raises(RuntimeError, match="bounded device wait expired"):
            call()
            lsa.check_status()  # without the checked mode
        wait_limit(-1)
        got = call()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    lsa.check_status()


def test_wait_limits_out_of_range_are_refused(lsa):
    from lsa_b200 import _lib

    assert _lib.lib().lsa_shared_prefix_wait_limit(10 ** 10 + 1) == _lib.ERR_ARG


def test_an_item_may_run_longer_than_a_wait(lsa, wait_limit):
    """The limit is one wait's. Whole row tiles of 1025 chunks run 1.7 ms or more with waits of a few us, and
    the warp that zeroes the last V tile's tail waits for all of them."""
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(BF)
    q, kp, vp, k, v = r(37, 64, 16, 128), r(131072, 4, 128), r(131072, 4, 128), r(37, 70, 4, 128), r(37, 70, 4, 128)
    lengths = torch.full((37,), 70, dtype=torch.int32, device=DEV)
    want = lsa.shared_prefix_attention(q, kp, vp, k, v, lengths)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    wait_limit(500_000)
    start.record()
    got = lsa.shared_prefix_attention(q, kp, vp, k, v, lengths)
    end.record()
    lsa.check_status()
    assert torch.equal(got, want) and start.elapsed_time(end) > 1.0


def reported():
    from lsa_b200 import _lib

    return {t.data_ptr(): t for t in _lib.torch_ops().workspace_counters()}


def small(lsa, seed=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(BF)
    return (r(30, 1, 8, 64), r(300, 2, 64), r(300, 2, 64), r(30, 40, 2, 64), r(30, 40, 2, 64),
            torch.full((30,), 40, dtype=torch.int32, device=DEV))


def read_rows(R):
    """A sparse read of R rows (and R * Hkv counters) with split lists."""
    from lsa_b200 import _lib

    g = torch.Generator(device=DEV)
    g.manual_seed(R)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(BF)
    q, k, v = r(1, R, 8, 64), r(1, 4096, 2, 64), r(1, 4096, 2, 64)
    ids = torch.randint(0, 4096, (R, 2116), generator=g, device=DEV, dtype=torch.int32)
    lengths = torch.full((R,), 2110, dtype=torch.int32, device=DEV)
    return lambda: _lib.torch_ops().sparse_read(q, k, v, ids, lengths, 0.125)


def test_the_status_word_outlives_larger_calls(lsa):
    """Whatever a captured call may write its status to is still reported after the stream's counters have grown."""
    args = small(lsa)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lsa.shared_prefix_attention(*args)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        lsa.shared_prefix_attention(*args)
    words = [p for p, t in reported().items() if t.numel() == 1]
    before = max(t.numel() for t in reported().values())
    with torch.cuda.stream(side):
        read_rows(before)()
    side.synchronize()
    assert len(words) >= 1 and set(words) <= set(reported())


def test_a_timeout_word_disturbs_no_other_operator(lsa, monkeypatch):
    """The word that an expired wait leaves (planted here) is no ticket of the sparse read."""
    from lsa_b200 import _lib

    lsa.shared_prefix_attention(*small(lsa))
    words = [t for t in reported().values() if t.numel() == 1]
    assert words
    read = read_rows(3)
    want = read()
    for w in words:
        w.fill_(_lib.ERR_TIMEOUT)
    got = read()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="bounded device wait expired"):
        lsa.check_status()
    lsa.check_status()


def test_a_first_call_inside_a_capture(tmp_path):
    """In a fresh process: the first call of all is captured. The word is zero before any replay, and a
    replay leaves an unread timeout in place."""
    import pathlib
    import subprocess
    import sys

    pkg = pathlib.Path(__file__).resolve().parents[1] / "latent-sparse-attention-rocm_b200"
    code = f"""
import sys; sys.path.insert(0, {str(pkg)!r})
import torch, lsa_b200
from lsa_b200 import _lib
_lib.torch_ops()
d = "cuda"
a = [torch.randn(4, 1, 8, 64, device=d).bfloat16(), *(torch.randn(300, 2, 64, device=d).bfloat16() for _ in range(2)),
     *(torch.randn(4, 40, 2, 64, device=d).bfloat16() for _ in range(2)),
     torch.full((4,), 40, dtype=torch.int32, device=d)]
junk = torch.full((1 << 22,), 77, dtype=torch.uint8, device=d)
del junk
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = lsa_b200.shared_prefix_attention(*a)
lsa_b200.check_status()
words = [t for t in _lib.torch_ops().workspace_counters()]
assert words and all(int(t.abs().sum()) == 0 for t in words)
for t in words: t[0] = _lib.ERR_TIMEOUT
g.replay(); torch.cuda.synchronize()
assert all(int(t[0]) == _lib.ERR_TIMEOUT for t in words)
try:
    lsa_b200.check_status()
    raise SystemExit("an unread timeout was wiped")
except RuntimeError as e:
    assert "expired" in str(e)
g.replay(); torch.cuda.synchronize()
assert torch.equal(out, lsa_b200.shared_prefix_attention(*a))
lsa_b200.check_status()
print("captured first")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("case", [(19, 64, 32, 8, 128, 10007, 100), (19, 70, 56, 8, 64, 5000, 90)],
                         ids=lambda c: "-".join(map(str, c)))
def test_few_split_tiles_beside_whole_ones(lsa, case):
    """148 whole tiles and four in many parts, numbered by tile; with seven heads a group a tile has rows of no one."""
    from test_gpu_shared_prefix import check_all, make

    check_all(lsa, make(*case, BF, seed=21), BF)


def call_entry(lsa, q, k, v, lengths, scores, out, scores_out):
    """lsa_shared_prefix_attention itself, without a prefix."""
    from lsa_b200 import _lib

    L = _lib.lib()
    B, Tq, Hq, D = q.shape
    T, Hkv = k.shape[1:3]
    st = (ctypes.c_int64 * 13)(*q.stride()[:3], D, D, D, D, *k.stride()[:3], *v.stride()[:3])
    nbytes = L.lsa_shared_prefix_scratch(_lib.BF16, B, Tq, Hq, Hkv, D, 0, T, 1)
    scratch = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=DEV)
    return L.lsa_shared_prefix_attention(_lib.ptr(q), None, None, _lib.ptr(k), _lib.ptr(v), _lib.BF16, st,
                                         _lib.ptr(lengths), B, Tq, Hq, Hkv, D, 0, T, D ** -0.5, _lib.ptr(out), None,
                                         _lib.ptr(scores), _lib.ptr(scores_out), _lib.ptr(scratch), nbytes,
                                         _lib.ptr(_lib.status_word(q.device)), _lib.stream_of(q))


def test_the_entry_without_rows_passes_the_scores_on(lsa):
    k = torch.randn(2, 40, 2, 64, device=DEV).to(BF)
    q = torch.empty(2, 0, 4, 64, dtype=BF, device=DEV)
    scores = torch.rand(2, 2, 40, device=DEV)
    got = torch.full_like(scores, -7.0)
    lengths = torch.tensor([40, 3], dtype=torch.int32, device=DEV)
    assert call_entry(lsa, q, k, k, lengths, scores, torch.empty_like(q), got) == 0
    assert torch.equal(got, scores)
    assert call_entry(lsa, q, k, k, lengths, got, torch.empty_like(q), got) == 0  # in place
    assert torch.equal(got, scores)


def test_scales_past_fp32_are_refused(lsa):
    """A scale whose product with log2(e) is no finite positive fp32 number has no answer."""
    q, k = torch.ones(1, 1, 2, 64, dtype=BF, device=DEV), torch.zeros(1, 8, 2, 64, dtype=BF, device=DEV)
    lengths = torch.tensor([8], device=DEV)
    for scale in (1e-50, 3e38, 1e300):
        with pytest.raises(ValueError, match="scale"):
            lsa.shared_prefix_attention(q, k[0], k[0], k, k, lengths, scale)
    assert (lsa.shared_prefix_attention(q, k[0], k[0], k, k, lengths, 2e38) == 0).all()


def test_a_step_refused_by_the_operator_undoes_its_eviction(lsa):
    """What the step itself does not look at - here a prefix that does not fit - is refused by the operator,
    after the eviction that the step was due; the cache is as before."""
    cache, r = budgeted(lsa)
    cache.step(r(3, 4, 4, 64), r(3, 4, 2, 64), r(3, 4, 2, 64))
    k, v, scores, lengths = cache.k, cache.v, cache.scores, cache.lengths.clone()
    cache.k_prefix = cache.v_prefix = r(10, 1, 64)
    with pytest.raises(ValueError):
        cache.step(r(3, 5, 4, 64), r(3, 5, 2, 64), r(3, 5, 2, 64))
    assert cache.k is k and cache.v is v and cache.scores is scores and torch.equal(cache.lengths, lengths)
    cache.k_prefix = cache.v_prefix = None
    cache.step(r(3, 4, 4, 64), r(3, 4, 2, 64), r(3, 4, 2, 64))  # fits without an eviction
    assert cache.k is k and torch.equal(cache.lengths, lengths + 4)
