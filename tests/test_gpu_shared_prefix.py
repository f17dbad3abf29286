"""Shared-prefix attention and scored attention on the GPU against the formula in 64 bits.

Tolerances, from the arithmetic: the logits are fp32 sums of D exact products, so a logit is
off by at most D 2^-24 sum|q k| scale (below 1e-4 for these inputs) and a weight by that
relative; 16-bit inputs round each weight once more to 16 bits before its product with v
(u = 2^-8 bf16, 2^-11 fp16) and the output once. So
  |out - exact| <= u |exact| + (u + 2e-4) sum p |v| + 1e-6   (u = 0 for fp32 inputs),
  |score - exact| <= 2e-4 weight + 2^-23 score.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def make(B, Tq, Hq, Hkv, D, P, T, dt, seed=0, lengths=None, amp=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    q = (r(B, Tq, Hq, D) * amp).to(dt)
    kp, vp, k, v = r(P, Hkv, D).to(dt), r(P, Hkv, D).to(dt), r(B, T, Hkv, D).to(dt), r(B, T, Hkv, D).to(dt)
    if lengths is None:
        lengths = torch.randint(min(Tq, T), T + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
    else:
        lengths = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    scores = torch.rand(B, Hkv, T, generator=g, device=DEV)
    return q, kp, vp, k, v, lengths, scores


def want(q, kp, vp, k, v, lengths, scale=None):
    """out, sum p |v|, lse, own weights [B, Hkv, T] in float64, a sequence and KV head at a time."""
    B, Tq, Hq, D = q.shape
    P, Hkv, _ = kp.shape
    T, G = k.shape[1], Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, Tq, Hq, D, dtype=torch.float64, device=DEV)
    absum, lse = torch.zeros_like(out), torch.full((B, Tq, Hq), -math.inf, dtype=torch.float64, device=DEV)
    weights = torch.zeros(B, Hkv, T, dtype=torch.float64, device=DEV)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), T)
        for h in range(Hkv):
            key = torch.cat([kp[:, h], k[b, :n, h]]).double()
            val = torch.cat([vp[:, h], v[b, :n, h]]).double()
            qq = q[b, :, h * G:(h + 1) * G].double().reshape(Tq * G, D)
            limit = (P + torch.arange(Tq, device=DEV) + n - Tq + 1).clamp(min=P).repeat_interleave(G)
            s = (qq @ key.T) * scale
            s = s.masked_fill(torch.arange(P + n, device=DEV)[None] >= limit[:, None], -math.inf)
            if P + n == 0:
                continue
            x = torch.logsumexp(s, -1)
            p = torch.exp(s - torch.where(x == -math.inf, torch.zeros_like(x), x)[:, None])
            out[b, :, h * G:(h + 1) * G] = (p @ val).view(Tq, G, D)
            absum[b, :, h * G:(h + 1) * G] = (p @ val.abs()).view(Tq, G, D)
            lse[b, :, h * G:(h + 1) * G] = x.view(Tq, G)
            weights[b, h, :n] = p[:, P:].sum(0)
    return out, absum, lse, weights


def check_out(got, out, absum, dt):
    bound = U[dt] * out.abs() + (U[dt] + 2e-4) * absum + 1e-6
    over = (got.double() - out).abs() - bound
    assert not torch.isnan(got).any() and float(over.max()) <= 0, f"worst {float(over.max())} over the bound"


def check_all(lsa, args, dt, scale=None):
    q, kp, vp, k, v, lengths, scores = args
    out, absum, lse, weights = want(q, kp, vp, k, v, lengths, scale)
    got, got_lse = lsa.shared_prefix_attention(q, kp, vp, k, v, lengths, scale, return_lse=True)
    assert got.shape == q.shape and got.dtype == q.dtype and got.is_contiguous()
    check_out(got, out, absum, dt)
    same = got_lse.double() - lse
    same = torch.where(lse == -math.inf, torch.where(got_lse == -math.inf, 0.0, math.inf).double(), same)
    assert float(same.abs().max()) <= 2e-4
    before = scores.clone()
    o2, s2 = lsa.scored_attention(q, k, v, lengths, scores, scale, k_prefix=kp, v_prefix=vp)
    check_out(o2, out, absum, dt)
    assert torch.equal(scores, before) and s2.shape == scores.shape
    if k.shape[1] == 0:
        return
    ref = scores.double() + weights
    assert float(((s2.double() - ref).abs() - 2e-4 * weights - 2.0 ** -23 * ref.abs()).max()) <= 0
    T = k.shape[1]
    past = torch.arange(T, device=DEV)[None, None] >= lengths.clamp(0, T)[:, None, None]
    assert torch.equal(s2[past.expand_as(s2)], scores[past.expand_as(s2)])


CASES = [
    # B, Tq, Hq, Hkv, D, P, T
    (1, 1, 8, 8, 128, 1, 1),
    (1, 1, 32, 8, 128, 2000, 300),
    (3, 1, 32, 8, 128, 129, 65),
    (4, 1, 6, 2, 64, 127, 33),       # 3 query heads to a KV head
    (5, 2, 28, 4, 128, 1000, 200),   # 7 to one, 70 prefix rows
    (16, 1, 64, 8, 128, 4097, 129),  # 128 prefix rows
    (40, 1, 32, 4, 64, 700, 500),    # 320 prefix rows
    (2, 5, 8, 2, 64, 513, 77),
    (2, 17, 16, 1, 128, 300, 150),   # 16 to one
    (1, 1, 64, 1, 128, 555, 700),    # 64 to one
    (2, 64, 32, 8, 128, 640, 512),
    (2, 130, 8, 4, 128, 200, 333),
    (1, 257, 6, 2, 64, 0, 400),
    (2, 32, 32, 8, 128, 0, 3000),    # rows that score a long cache
    (1, 1, 32, 8, 128, 0, 20000),
    (2, 3, 5, 1, 64, 0, 128),
    (7, 4, 4, 1, 128, 256, 4),       # caches that hold the call's tokens alone
    (40, 64, 16, 4, 128, 300, 130),  # more row tiles than SMs: whole ones, and a split rest
    (1, 1030, 8, 2, 128, 260, 1500), # a long chunk: row tiles of one sequence, causal ranges of their own
    (3, 7, 8, 2, 64, 100, 0),        # no own cache at all
    (30, 1, 32, 8, 128, 900, 0),
    (2, 70, 16, 4, 128, 300, 0),
    (25, 150, 12, 3, 64, 200, 160),  # 600 rows a sequence, 75 of them in the last tile of three
]


@pytest.mark.parametrize("dt", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_against_64_bits(lsa, case, dt):
    check_all(lsa, make(*case, dt, seed=sum(case)), dt)


@pytest.mark.parametrize("dt", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("P", [0, 300])
@pytest.mark.parametrize("Tq", [1, 6, 40])
def test_rows_without_keys_and_odd_lengths(lsa, dt, P, Tq):
    """Lengths of zero, one, fewer than the call's rows, past the cache, negative: a row whose
    mask leaves nothing reads as zeros with log-sum-exp -inf."""
    lengths = [0, 1, Tq - 1, Tq, 128, 129, 140, 1000, -3]
    args = make(9, Tq, 8, 2, 128, P, 140, dt, seed=3, lengths=lengths)
    check_all(lsa, args, dt)
    if P == 0:
        out, lse = lsa.shared_prefix_attention(*args[:6], return_lse=True)
        assert (out[0] == 0).all() and (lse[0] == -math.inf).all() and (out[8] == 0).all()


@pytest.mark.parametrize("dt", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Tq,Hq,T", [(1, 8, 300), (8, 8, 300), (48, 16, 300), (1, 32, 64)])
def test_unwritten_slots_are_never_used(lsa, dt, Tq, Hq, T):
    """NaN, infinities and the type's lowest value past the lengths change no bit."""
    lengths = [Tq, Tq + 1, 100, 129, T - 1, T] if T > 200 else [1, 2, 31, 33, 63, 64]
    q, kp, vp, k, v, lengths, scores = make(6, Tq, Hq, 2, 128, 70, T, dt, seed=5, lengths=lengths)
    clean = lsa.scored_attention(q, k, v, lengths, scores, k_prefix=kp, v_prefix=vp)
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(dt).min):
        k2, v2 = k.clone(), v.clone()
        for b in range(6):
            k2[b, int(lengths[b]):], v2[b, int(lengths[b]):] = bad, bad
        got = lsa.scored_attention(q, k2, v2, lengths, scores, k_prefix=kp, v_prefix=vp)
        assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])


@pytest.mark.parametrize("dt", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Tq,B,P", [(1, 3, 40), (1, 30, 400), (40, 3, 0), (70, 2, 300)])
def test_a_nan_query_stays_in_its_row(lsa, dt, Tq, B, P):
    """A NaN row gives NaN outputs, and no other row's bits change."""
    q, kp, vp, k, v, lengths, scores = make(B, Tq, 8, 2, 128, P, 100, dt, seed=6)
    clean = lsa.shared_prefix_attention(q, kp, vp, k, v, lengths)
    q2 = q.clone()
    q2[B - 1, Tq - 1, 5] = math.nan
    got, lse = lsa.shared_prefix_attention(q2, kp, vp, k, v, lengths, return_lse=True)
    assert torch.isnan(got[B - 1, Tq - 1, 5]).all() and torch.isnan(lse[B - 1, Tq - 1, 5])
    got[B - 1, Tq - 1, 5] = clean[B - 1, Tq - 1, 5]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("Tq,B", [(1, 3), (16, 3), (1, 70)])
def test_strided_views(lsa, dt, Tq, B):
    """Head-major caches, a query cut from a fused projection, a prefix cut from a longer one:
    the same bits as their contiguous copies."""
    Hq, Hkv, D, P, T = 8, 2, 128, 333, 150
    q, kp, vp, k, v, lengths, scores = make(B, Tq, Hq, Hkv, D, P, T, dt, seed=7)
    fused = torch.randn(B, Tq, Hq + 2 * Hkv, D, device=DEV).to(dt)
    fused[:, :, :Hq] = q
    k2 = k.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    v2 = torch.cat([v, v], -1)[..., :D]
    kp2 = torch.cat([kp, kp])[:P]
    vp2 = vp.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    a = lsa.scored_attention(q, k, v, lengths, scores, k_prefix=kp, v_prefix=vp)
    b = lsa.scored_attention(fused[:, :, :Hq], k2, v2, lengths, scores, k_prefix=kp2, v_prefix=vp2)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # rows off the 16-byte boundaries, and a transposed head dimension, are copied
    off = torch.empty(B * T * Hkv * D + 1, dtype=dt, device=DEV)[1:].view(B, T, Hkv, D)
    off.copy_(k)
    c = lsa.scored_attention(q, off, v.transpose(2, 3).contiguous().transpose(2, 3), lengths, scores, k_prefix=kp,
                             v_prefix=vp)
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


@pytest.mark.parametrize("dt", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Tq", [1, 24])
def test_large_logits_and_scale(lsa, dt, Tq):
    """Logits of several tens, a few keys holding all the weight, and a scale of one's own. The
    logits' error grows with them, so the rows are held to a bound of their own size."""
    q, kp, vp, k, v, lengths, scores = make(4, Tq, 16, 4, 64, 900, 260, dt, seed=9, amp=6.0)
    out, absum, _, weights = want(q, kp, vp, k, v, lengths, 0.2)
    got, s2 = lsa.scored_attention(q, k, v, lengths, scores, 0.2, k_prefix=kp, v_prefix=vp)
    check_out(got, out, absum, dt)
    ref = scores.double() + weights
    # |logit| error <= D 2^-24 sum|q k| scale: with |q| ~ 6, 64 terms, below 6e-4
    assert float(((s2.double() - ref).abs() - 6e-4 * weights - 2.0 ** -23 * ref).max()) <= 0


def test_prefix_equals_copies_in_every_cache(lsa):
    """The prefix read once gives what each sequence would read from its own copy."""
    q, kp, vp, k, v, lengths, _ = make(20, 1, 32, 8, 128, 800, 100, BF, seed=11)
    a = lsa.shared_prefix_attention(q, kp, vp, k, v, lengths)
    whole_k = torch.cat([kp[None].expand(20, -1, -1, -1), k], 1)
    whole_v = torch.cat([vp[None].expand(20, -1, -1, -1), v], 1)
    b = lsa.shared_prefix_attention(q, kp[:0], vp[:0], whole_k, whole_v, lengths + 800)
    assert float((a.float() - b.float()).abs().max()) <= 2e-2


@pytest.mark.parametrize("Tq", [1, 40])
def test_tiny_scales(lsa, Tq):
    """All weights equal in the limit: the mean of the visible values."""
    q, kp, vp, k, v, lengths, scores = make(2, Tq, 8, 2, 128, 90, 140, BF, seed=12, lengths=[140, 77])
    for scale in (1e-30, 1e-44):
        out, absum, _, _ = want(q, kp, vp, k, v, lengths, scale)
        check_out(lsa.shared_prefix_attention(q, kp, vp, k, v, lengths, scale), out, absum, BF)


def test_refusals(lsa):
    q, kp, vp, k, v, lengths, scores = make(2, 1, 8, 2, 128, 16, 32, BF)
    bad = [(q.float(), kp, vp, k, v, lengths), (q, kp[:, :1], vp[:, :1], k, v, lengths), (q, kp, vp[:8], k, v, lengths),
           (q, kp, vp, k, v[:, :8], lengths), (q[:1], kp, vp, k, v, lengths), (q, kp, vp, k, v, lengths[:1]),
           (q, kp, vp, k, v, lengths.float()), (q[:, :, :7], kp, vp, k, v, lengths), (q[0], kp, vp, k, v, lengths),
           (q[..., :32], kp[..., :32], vp[..., :32], k[..., :32], v[..., :32], lengths),
           (q, kp, vp, k.cpu(), v, lengths), (q, kp, vp, k, v, lengths.cpu())]
    for args in bad:
        with pytest.raises(ValueError):
            lsa.shared_prefix_attention(*args)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            lsa.shared_prefix_attention(q, kp, vp, k, v, lengths, scale)
    for s in (scores[:, :1], scores.double(), scores[:, :, :8], scores[0]):
        with pytest.raises(ValueError, match="scores"):
            lsa.scored_attention(q, k, v, lengths, s)
    with pytest.raises(ValueError, match="prefix"):
        lsa.scored_attention(q, k, v, lengths, scores, v_prefix=vp)
    for kw in (dict(budget=-1), dict(budget=10, window_size=8, sink_size=4), dict(budget=20, window_size=8, capacity=10),
               dict(budget=20, window_size=-1), dict(budget=20, window_size=4, sink_size=-1)):
        with pytest.raises(ValueError):
            lsa.evict(k, v, scores, lengths, **kw)
    with pytest.raises(ValueError, match="16 bytes"):
        lsa.evict(k[..., :4].contiguous(), v[..., :4].contiguous(), scores, lengths, 20, 4)
    empty = lsa.shared_prefix_attention(q[:0], kp, vp, k[:0], v[:0], lengths[:0])
    assert empty.shape == (0, 1, 8, 128)


def test_same_bits_every_time(lsa):
    for case in [(16, 1, 32, 8, 128, 5000, 600), (4, 40, 32, 8, 128, 1000, 600), (1, 1, 32, 8, 128, 0, 30000)]:
        args = make(*case, BF, seed=13)
        first = lsa.scored_attention(args[0], args[3], args[4], args[5], args[6], k_prefix=args[1], v_prefix=args[2])
        for _ in range(3):
            again = lsa.scored_attention(args[0], args[3], args[4], args[5], args[6], k_prefix=args[1],
                                         v_prefix=args[2])
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("case", [(4, 1, 32, 8, 128, 1000, 200), (3, 40, 16, 4, 128, 500, 300)],
                         ids=["decode", "chunk"])
def test_other_stream_and_graph(lsa, case):
    """On a stream of its own, and captured once and replayed on new inputs."""
    args = make(*case, BF, seed=15)
    new = make(*case, BF, seed=16)
    call = lambda a: lsa.scored_attention(a[0], a[3], a[4], a[5], a[6], k_prefix=a[1], v_prefix=a[2])
    want1, want2 = call(args), call(new)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(args)
    side.synchronize()
    assert torch.equal(got[0], want1[0]) and torch.equal(got[1], want1[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = call(args)
    for x, y in zip(args, new):
        x.copy_(y)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want2[0]) and torch.equal(got[1], want2[1])
    lsa.check_status()


def test_a_larger_call_leaves_a_captured_graph_alone(lsa):
    """A captured call replays the same bits after larger eager calls on its stream and after what
    they freed has been written over."""
    args = make(4, 1, 32, 8, 128, 1000, 200, BF, seed=18)
    call = lambda a: lsa.scored_attention(a[0], a[3], a[4], a[5], a[6], k_prefix=a[1], v_prefix=a[2])
    expect = [x.clone() for x in call(args)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(args)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = call(args)
    big = make(24, 33, 32, 8, 128, 2000, 900, BF, seed=19)
    with torch.cuda.stream(side):
        for _ in range(2):
            call(big)
        junk = [torch.full((1 << 22,), 255, dtype=torch.uint8, device=DEV) for _ in range(64)]
        graph.replay()
        same = [bool((x == 255).all()) for x in junk]
    side.synchronize()
    assert torch.equal(got[0], expect[0]) and torch.equal(got[1], expect[1]) and all(same)


@pytest.mark.parametrize("Hq,own", [(8, False), (128, False), (8, True), (128, True)])
def test_offsets_past_32_bits(lsa, Hq, own):
    """A cache of more than 2^31 elements: the last keys hold the weight."""
    n, Hkv, D = (1 << 21) + 300, 8, 128
    assert n * Hkv * D > 1 << 31
    k = torch.zeros(n, Hkv, D, dtype=BF, device=DEV)
    v = torch.zeros(n, Hkv, D, dtype=BF, device=DEV)
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    k[-200:], v[-200:] = (torch.randn(200, Hkv, D, generator=g, device=DEV).to(BF) for _ in range(2))
    q = torch.randn(1, 1, Hq, D, generator=g, device=DEV).to(BF) * 8
    if own:
        args = (q, k[:0], v[:0], k[None], v[None], torch.tensor([n], device=DEV))
    else:
        args = (q, k, v, k[None, :1], v[None, :1], torch.tensor([0], device=DEV))
    got = lsa.shared_prefix_attention(*args)
    # the zero keys have logit 0 and value 0: they enter the sum alone
    s = torch.einsum("hgd,jhd->hgj", q[0, 0].view(Hkv, Hq // Hkv, D).double(), k[-200:].double()) * D ** -0.5
    e = torch.exp(s)
    total = e.sum(-1, keepdim=True) + (n - 200)
    out = torch.einsum("hgj,jhd->hgd", e / total, v[-200:].double()).reshape(1, 1, Hq, D)
    absum = torch.einsum("hgj,jhd->hgd", e / total, v[-200:].double().abs()).reshape(1, 1, Hq, D)
    check_out(got, out, absum, BF)


def test_compiles_as_one_node(lsa):
    args = make(2, 1, 8, 2, 128, 100, 50, BF, seed=17)
    from lsa_b200 import _lib

    ops = _lib.torch_ops()
    fn = torch.compile(lambda *a: ops.shared_prefix_attention(*a, 0.1), backend="eager", fullgraph=True)
    assert torch.equal(fn(*args[:6]), ops.shared_prefix_attention(*args[:6], 0.1))
