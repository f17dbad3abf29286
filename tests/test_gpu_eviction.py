"""Eviction on the GPU against a numpy selection: ids, copies and counts equal exactly.

The serving loop under a shared prefix - attend, score, append, evict - is checked against the
same loop in 64 bits that starts each step from the GPU's own state."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def want_ids(scores, n, budget, window, sink):
    """One row's kept ids: the order of the scores' bits (as integers), ties to the lower index."""
    if n <= budget:
        return np.arange(n)
    bits = scores[:n].view(np.int32).astype(np.int64)
    order = np.where(bits >= 0, bits, bits ^ 0x7FFFFFFF)
    mid = np.arange(sink, n - window)
    best = mid[np.lexsort((mid, -order[mid]))][:budget - sink - window]
    return np.sort(np.concatenate([np.arange(sink), best, np.arange(n - window, n)]))


def check(lsa, k, v, scores, lengths, budget, window, sink, capacity=None):
    e = lsa.evict(k, v, scores, lengths, budget, window_size=window, sink_size=sink, capacity=capacity)
    B, T, Hkv, D = k.shape
    C = budget if capacity is None else capacity
    assert e.k.shape == e.v.shape == (B, C, Hkv, D) and e.k.dtype == k.dtype
    assert e.scores.shape == e.ids.shape == (B, Hkv, C)
    n = lengths.cpu().numpy().clip(0, T)
    assert np.array_equal(e.lengths.cpu().numpy(), np.minimum(n, budget))
    sc = scores.cpu().numpy()
    ids = np.full((B, Hkv, C), -1, np.int32)
    for b in range(B):
        for h in range(Hkv):
            w = want_ids(sc[b, h], int(n[b]), budget, window, sink)
            ids[b, h, :len(w)] = w
    assert np.array_equal(e.ids.cpu().numpy(), ids)
    at = torch.from_numpy(ids).to(DEV).long()
    dead = at < 0
    at = at.clamp(min=0)
    if T and C:
        bits = lambda t: t.contiguous().view(torch.uint8)
        rows = at.permute(0, 2, 1)[..., None].expand(B, C, Hkv, D)
        for got, src in ((e.k, k), (e.v, v)):
            ref = torch.gather(src, 1, rows).masked_fill(dead.permute(0, 2, 1)[..., None], 0)
            assert torch.equal(bits(got), bits(ref))
        ref = torch.gather(scores, 2, at).masked_fill(dead, 0)
        assert torch.equal(bits(e.scores), bits(ref))
    return e


def make(B, T, Hkv, D, dt, seed, levels=None):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    k, v = (torch.randn(B, T, Hkv, D, generator=g, device=DEV).to(dt) for _ in range(2))
    s = torch.rand(B, Hkv, T, generator=g, device=DEV)
    if levels:
        s = (s * levels).floor() / levels
    return k, v, s


@pytest.mark.parametrize("T,budget,window,sink", [
    (1, 1, 0, 0), (1, 0, 0, 0), (2, 1, 0, 1), (2, 1, 1, 0), (33, 32, 8, 2), (100, 7, 3, 4), (1023, 1000, 64, 4),
    (1025, 512, 0, 0), (2112, 2048, 64, 4), (5000, 100, 1, 0), (9001, 4096, 256, 1), (40000, 3001, 64, 4),
    (70001, 66000, 64, 4),
])
@pytest.mark.parametrize("levels", [None, 3])
def test_ids_and_copies(lsa, T, budget, window, sink, levels):
    k, v, s = make(3, T, 2, 64, BF, T + budget, levels)
    lengths = torch.tensor([T, max(T - 5, 0), T // 2], dtype=torch.int32, device=DEV)
    check(lsa, k, v, s, lengths, budget, window, sink)
    check(lsa, k, v, s, lengths, budget, window, sink, capacity=budget + 37)


def test_one_long_cache(lsa):
    k, v, s = make(1, 300001, 1, 64, BF, 3, 1000)
    check(lsa, k, v, s, torch.tensor([300001], device=DEV), 8192, 256, 4)
    check(lsa, k, v, s, torch.tensor([260000], device=DEV), 250001, 256, 4)


def test_lengths_zero_one_and_past_the_cache(lsa):
    k, v, s = make(7, 130, 3, 128, HF, 4)
    lengths = torch.tensor([0, 1, 64, 65, 130, 500, -2], dtype=torch.int64, device=DEV)
    check(lsa, k, v, s, lengths, 64, 16, 4)
    check(lsa, k, v, s, lengths, 64, 60, 4)  # sinks and window fill the budget
    check(lsa, k, v, s, lengths, 0, 0, 0, capacity=5)
    check(lsa, k[:, :0], v[:, :0], s[:, :, :0], lengths, 16, 4, 4)


@pytest.mark.parametrize("T", [200, 5000])
def test_order_of_special_scores(lsa, T):
    """NaNs of both signs, infinities, zeros of both signs, subnormals and equal runs."""
    k, v, s = make(2, T, 2, 64, BF, 5, 4)
    bits = s.view(torch.int32)
    special = [0x7FC00000, -0x400000, 0x7F800000, -0x800000, 0, -(1 << 31), 1, -(1 << 31) + 1, 0x7F7FFFFF, -0x800001]
    for i, x in enumerate(special):
        bits[:, :, 10 + 3 * i] = x
        bits[:, :, 90 + i] = x
    lengths = torch.tensor([T, T - 1], dtype=torch.int32, device=DEV)
    for budget in (12, 21, 40, 90, T - 10, T - 1):
        check(lsa, k, v, s, lengths, budget, 5, 3)
    s.fill_(0.25)  # every key level
    check(lsa, k, v, s, lengths, 77, 8, 4)
    check(lsa, k, v, s, lengths, T - 2, 8, 4)


@pytest.mark.parametrize("dt,D", [(F32, 64), (HF, 80), (BF, 24), (torch.uint8, 16), (BF, 192)])
def test_row_sizes_and_types(lsa, dt, D):
    k, v, s = make(2, 777, 2, D, F32, 6)
    k, v = ((x * 40).to(dt) if dt == torch.uint8 else x.to(dt) for x in (k.abs(), v.abs()))
    check(lsa, k, v, s, torch.tensor([777, 300], device=DEV), 333, 32, 4)


def test_strided_caches_and_payload_bits(lsa):
    """Head-major caches and views of a longer one; rows are copied as bytes, NaN among them."""
    k, v, s = make(2, 900, 4, 128, BF, 8)
    k[0, 5, 1, 3] = float("nan")
    k2 = k.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    v2 = torch.cat([v, v], 1)[:, :900]
    s2 = torch.cat([s, s], 2)[:, :, :900]
    lengths = torch.tensor([900, 640], dtype=torch.int32, device=DEV)
    check(lsa, k2, v2, s2, lengths, 256, 16, 6)


def test_offsets_past_32_bits(lsa):
    T, Hkv, D = (1 << 21) + 300, 8, 128
    k = torch.zeros(1, T, Hkv, D, dtype=BF, device=DEV)
    k[0, :, :, 0] = (torch.arange(T, device=DEV) % 251)[:, None].to(BF)
    s = torch.zeros(1, Hkv, T, device=DEV)
    s[:, :, -150:] = 1.0
    e = lsa.evict(k, k, s, torch.tensor([T], device=DEV), 100, window_size=10, sink_size=2)
    ids = torch.cat([torch.tensor([0, 1], device=DEV), torch.arange(T - 150, T - 62, device=DEV),
                     torch.arange(T - 10, T, device=DEV)]).int()
    assert torch.equal(e.ids, ids[None, None].expand(1, Hkv, -1))
    assert torch.equal(e.k[0, :, 3], k[0, ids.long(), 3])


def test_other_stream_and_graph(lsa):
    a, b = make(4, 1500, 2, 128, BF, 10), make(4, 1500, 2, 128, BF, 11)
    lengths = torch.tensor([1500, 900, 400, 1], dtype=torch.int32, device=DEV)
    w1 = lsa.evict(*a, lengths, 500, 64, 4)
    w2 = lsa.evict(*b, lengths, 500, 64, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = lsa.evict(*a, lengths, 500, 64, 4)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, w1))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = lsa.evict(*a, lengths, 500, 64, 4)
    for x, y in zip(a, b):
        x.copy_(y)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, w2))


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Tq,P", [(1, 500), (3, 0)])
def test_serving_loop(lsa, dt, Tq, P):
    """The whole loop: every step's output and scores against the formula in 64 bits on the state
    that the step started from, through several evictions. Tolerances as in the attention's tests."""
    B, Hq, Hkv, D, T, budget, room = 3, 8, 2, 128, 150, 96, 7
    g = torch.Generator(device=DEV)
    g.manual_seed(Tq)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dt)
    kp, vp = (r(P, Hkv, D), r(P, Hkv, D)) if P else (None, None)
    cache = lsa.BudgetedCache(r(B, T, Hkv, D), r(B, T, Hkv, D), [150, 96, 20], budget, room, window_size=16,
                              sink_size=4, k_prefix=kp, v_prefix=vp, scores=torch.rand(B, Hkv, T, device=DEV))
    assert cache.lengths.tolist() == [96, 96, 20] and cache.k.shape[1] == budget + room
    u = 2.0 ** -8 if dt == BF else 0.0
    evictions = 0
    for _ in range(20):
        before = [int(n) for n in cache.lengths]
        q, k_new, v_new = r(B, Tq, Hq, D), r(B, Tq, Hkv, D), r(B, Tq, Hkv, D)
        old = cache.scores
        out = cache.step(q, k_new, v_new)
        after = [int(n) for n in cache.lengths]
        evicted = after[0] != before[0] + Tq
        evictions += evicted
        assert after == [min(n, budget if evicted else n) + Tq for n in before]
        for b in range(B):
            n = after[b]
            assert torch.equal(cache.k[b, n - Tq:n], k_new[b]) and torch.equal(cache.v[b, n - Tq:n], v_new[b])
            for h in range(Hkv):
                key, val = cache.k[b, :n, h].double(), cache.v[b, :n, h].double()
                if P:
                    key, val = torch.cat([kp[:, h].double(), key]), torch.cat([vp[:, h].double(), val])
                s = torch.einsum("tgd,jd->tgj", q[b, :, 4 * h:4 * h + 4].double(), key) * D ** -0.5
                last = P + n - Tq + torch.arange(Tq, device=DEV)
                s = s.masked_fill(torch.arange(P + n, device=DEV) > last[:, None, None], -float("inf"))
                p = torch.softmax(s, -1)
                want, absum = p @ val, p @ val.abs()
                assert float(((out[b, :, 4 * h:4 * h + 4].double() - want).abs() - u * want.abs()
                              - (u + 2e-4) * absum - 1e-6).max()) <= 0
                if not evicted:
                    w = p[..., P:].sum((0, 1))
                    assert float(((cache.scores[b, h, :n].double() - old[b, h, :n].double() - w).abs()
                                  - 2e-4 * w - 2.0 ** -22 * (old[b, h, :n] + 1)).max()) <= 0
    assert evictions >= 2
    with pytest.raises(ValueError, match="room"):
        cache.step(r(B, 8, Hq, D), r(B, 8, Hkv, D), r(B, 8, Hkv, D))
    lsa.check_status()
