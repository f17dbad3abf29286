"""Norms and rotation on a B200 against their definition in 64 bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def plain(x, positions, f, weight, eps, interleaved, amplitude):
    """(output, how far off a kernel may be), 64 bits on the CPU.

    fp32: the mean of D squares, its root, two products and the rotation's two products and sum are at most D + 16
    roundings of 2^-24 of the pair's magnitudes (some fifteen of them in earnest: the mean's error is halved by the root
    and its additions are pairwise; the others leave room for the special-function unit's sine and cosine of 16-bit
    values, 2^-21); sine and cosine of fp32 values 2^-22 with the rounding of the reduced angle, 2^-26 of a turn; the
    output is rounded once."""
    y = x.double()
    D, R = y.shape[-1], 2 * f.numel()
    if weight is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * weight.double()
    angle = (positions.double()[..., None] * f.double())[:, :, None]
    cos, sin = angle.cos() * amplitude, angle.sin() * amplitude
    out, size = y.clone(), y.abs()
    i = torch.arange(R // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    out[..., a], out[..., b] = y[..., a] * cos - y[..., b] * sin, y[..., a] * sin + y[..., b] * cos
    both = (y[..., a].abs() + y[..., b].abs()) * max(1.0, abs(amplitude))
    size[..., a], size[..., b] = both, both
    off = torch.finfo(x.dtype).eps / 2 * out.abs() + ((D + 16) * 2.0 ** -24 + 2.0 ** -22) * size
    return out, off + torch.finfo(x.dtype).smallest_normal * 2.0 ** -7


def check(got, want, off):
    assert not bool(((got.double().cpu() - want).abs() > off).any()), float(((got.double().cpu() - want).abs() / off).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,Hq,Hkv,D,R,norm", [
    (1, 1, 1, 1, 64, 64, True), (3, 1, 32, 8, 128, 128, True), (2, 5, 3, 1, 256, 256, True), (1, 33, 7, 7, 128, 32, False),
    (2, 17, 8, 2, 64, 16, True), (1, 4, 5, 2, 256, 0, True), (5, 3, 1, 2, 128, 112, False), (1, 700, 6, 2, 128, 64, True)])
def test_norm_rotate(lsa, dtype, interleaved, B, T, Hq, Hkv, D, R, norm):
    g = torch.Generator().manual_seed(1)
    q, k = (torch.randn(B, T, h, D, generator=g).to(dtype) for h in (Hq, Hkv))
    q[0, 0] *= 1000.0
    k[0, 0] = 0.0
    qw = (torch.randn(D, generator=g) + 1).to(dtype) if norm else None
    kw = torch.randn(D, generator=g) + 1 if norm else None  # fp32 weights beside 16-bit values
    f, amplitude = lsa.rotary_frequencies(R, 10000.0) if R else (torch.empty(0, dtype=torch.float64), 1.0)
    pos = torch.randint(0, 1 << 20, (B, T), generator=g)
    pos[0, 0] = 0
    pos[-1, -1] = (1 << 26) - 1
    cu = [None if t is None else t.cuda() for t in (qw, kw)]
    a, b = lsa.norm_rotate(q.cuda(), k.cuda(), pos.cuda(), f.cuda(), *cu, interleaved=interleaved, amplitude=1.3)
    assert a.dtype == dtype and a.shape == q.shape and b.shape == k.shape and a.is_contiguous() and b.is_contiguous()
    check(a, *plain(q, pos, f, qw, 1e-6, interleaved, 1.3))
    check(b, *plain(k, pos, f, kw, 1e-6, interleaved, 1.3))


def test_strides_shared_positions_and_one_weight(lsa):
    """Slices of a joint projection (not copied), positions of one sequence for all, int32 and negative ones, a
    weight for the keys alone, frequencies in fp32."""
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(3, 9, 12, 128, generator=g).to(torch.bfloat16)
    kw = torch.randn(128, generator=g).to(torch.bfloat16)
    f, _ = lsa.rotary_frequencies(128, 1e6, "linear", 4.0)
    f = f.float()
    pos = torch.arange(-4, 5, dtype=torch.int32)
    on = qkv.cuda()
    wide = torch.stack([pos, pos], -1).cuda()
    for p in (pos.cuda(), wide[:, 0], pos.long().cuda().expand(3, 9)):
        a, b = lsa.norm_rotate(on[:, :, :8], on[:, :, 8:10], p, f.cuda(), None, kw.cuda(), eps=1e-3)
        check(a, *plain(qkv[:, :, :8], pos.expand(3, 9), f, None, 1e-3, False, 1.0))
        check(b, *plain(qkv[:, :, 8:10], pos.expand(3, 9), f, kw, 1e-3, False, 1.0))
    turned = on.transpose(2, 3).contiguous().transpose(2, 3)  # a head's values apart: copied
    a, _ = lsa.norm_rotate(turned[:, :, :8], turned[:, :, 8:10], pos.cuda(), f.cuda())
    check(a, *plain(qkv[:, :, :8], pos.expand(3, 9), f, None, 1e-6, False, 1.0))


def test_head_of_nan_stays_its_own(lsa):
    g = torch.Generator().manual_seed(3)
    q, k = (torch.randn(1, 3, 4, 64, generator=g) for _ in range(2))
    f, _ = lsa.rotary_frequencies(64)
    w = torch.ones(64)
    pos = torch.arange(3)
    want, off = plain(q, pos[None], f, w, 1e-6, False, 1.0)
    q[0, 1, 2, 7] = math.nan
    a, _ = lsa.norm_rotate(q.cuda(), k.cuda(), pos.cuda(), f.cuda(), w.cuda(), w.cuda())
    keep = torch.ones(1, 3, 4, dtype=torch.bool)
    keep[0, 1, 2] = False
    assert a.cpu()[0, 1, 2].isnan().all()
    check(a.cpu()[keep], want[keep], off[keep])


def test_empty_stream_and_graph(lsa):
    f, _ = lsa.rotary_frequencies(64)
    a, b = lsa.norm_rotate(torch.empty(0, 4, 2, 64, device="cuda"), torch.empty(0, 4, 1, 64, device="cuda"),
                           torch.arange(4, device="cuda"), f.cuda())
    assert a.shape == (0, 4, 2, 64) and b.shape == (0, 4, 1, 64)
    q, k = torch.randn(2, 6, 4, 64, device="cuda"), torch.randn(2, 6, 2, 64, device="cuda")
    pos, f = torch.arange(6, device="cuda"), f.cuda()
    want = lsa.norm_rotate(q, k, pos, f)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = lsa.norm_rotate(q, k, pos, f)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = lsa.norm_rotate(q, k, pos, f)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(want, again, out))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_infinities_that_do_not_turn_stay_their_own(lsa, dtype, interleaved):
    """Without a norm every value past the first R leaves as it came, whatever lies beside it."""
    g = torch.Generator().manual_seed(4)
    q, k = (torch.randn(1, 2, 3, 128, generator=g).to(dtype) for _ in range(2))
    q[0, 0, 0, 32], q[0, 1, 2, 127], q[0, 1, 1, 77] = math.inf, -math.inf, math.nan
    f, _ = lsa.rotary_frequencies(32)
    a, b = lsa.norm_rotate(q.cuda(), k.cuda(), torch.arange(2).cuda(), f.cuda(), interleaved=interleaved)
    assert torch.equal(a.cpu()[..., 32:].nan_to_num(7.0), q[..., 32:].nan_to_num(7.0)) and torch.equal(b.cpu()[..., 32:], k[..., 32:])
    assert bool(a.cpu()[..., :32].isfinite().all()) and bool((a.cpu().isnan() == q.isnan()).all())
