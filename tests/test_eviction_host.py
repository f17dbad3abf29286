"""Refusals and shapes of the shared-prefix attention, the scored attention and the eviction,
without a GPU."""

import ctypes

import pytest
import torch

import lsa_b200
from lsa_b200 import _lib


def _prefix_args(device, B=2, Tq=1, Hq=8, Hkv=2, D=128, P=16, T=8, dt=torch.bfloat16):
    e = lambda *s: torch.empty(*s, dtype=dt, device=device)
    return [e(B, Tq, Hq, D), e(P, Hkv, D), e(P, Hkv, D), e(B, T, Hkv, D), e(B, T, Hkv, D),
            torch.empty(B, dtype=torch.int32, device=device)]


def test_meta_shapes():
    ops = _lib.torch_ops()
    a = _prefix_args("meta", Tq=3)
    out, lse = ops.shared_prefix_attention_lse(*a, 0.1)
    assert ops.shared_prefix_attention(*a, 0.1).shape == a[0].shape
    assert out.shape == a[0].shape and out.dtype == a[0].dtype
    assert lse.shape == (2, 3, 8) and lse.dtype == torch.float32
    s = torch.empty(2, 2, 8, device="meta")
    out, s2 = ops.scored_attention(a[0], a[3], a[4], a[5], s, 0.1, a[1], a[2])
    assert out.shape == a[0].shape and s2.shape == s.shape
    k, v, s2, n, ids = ops.evict(a[3], a[4], s, a[5], 4, 1, 1, 6)
    assert k.shape == v.shape == (2, 6, 2, 128) and s2.shape == ids.shape == (2, 2, 6) and n.shape == (2,)
    assert n.dtype == ids.dtype == torch.int32


def test_cpu_tensors_are_refused():
    a = _prefix_args("cpu")
    with pytest.raises(ValueError, match="CUDA"):
        lsa_b200.shared_prefix_attention(*a)
    with pytest.raises(ValueError, match="CUDA"):
        lsa_b200.scored_attention(a[0], a[3], a[4], a[5], torch.zeros(2, 2, 8))
    with pytest.raises(ValueError, match="CUDA"):
        lsa_b200.evict(a[3], a[4], torch.zeros(2, 2, 8), a[5], 4, 1, 1)


def test_half_a_prefix_is_refused():
    a = _prefix_args("cpu")
    with pytest.raises(ValueError, match="prefix"):
        lsa_b200.scored_attention(a[0], a[3], a[4], a[5], torch.zeros(2, 2, 8), k_prefix=a[1])


def _lib_or_skip():
    try:
        return _lib.lib()
    except OSError as e:
        pytest.skip(f"CUDA runtime not loadable here: {e}")


def test_c_entries_refuse_before_any_cuda_call():
    """Sizes, alignments and missing buffers that no kernel takes return LSA_ERR_ARG."""
    L = _lib_or_skip()
    buf = ctypes.c_void_p(4096)  # never dereferenced
    ok = dict(q=buf, kp=buf, vp=buf, k=buf, v=buf, dtype=2, strides=[1024, 1024, 128] + [256, 128] * 2 + [2048, 256, 128] * 2,
              lengths=buf, B=2, Tq=1, Hq=8, Hkv=2, D=128, P=16, T=8, scale=0.1, out=buf, lse=None, scores=None,
              scores_out=None, scratch=buf, bytes=1 << 30, status=buf)

    def call(**kw):
        a = dict(ok, **kw)
        st = None if a["strides"] is None else (ctypes.c_int64 * 13)(*a["strides"])
        return L.lsa_shared_prefix_attention(a["q"], a["kp"], a["vp"], a["k"], a["v"], a["dtype"], st, a["lengths"],
                                             a["B"], a["Tq"], a["Hq"], a["Hkv"], a["D"], a["P"], a["T"], a["scale"],
                                             a["out"], a["lse"], a["scores"], a["scores_out"], a["scratch"],
                                             a["bytes"], a["status"], None)

    for kw in (dict(D=96), dict(Hq=7), dict(Hq=130, Hkv=2), dict(Hkv=0), dict(dtype=3), dict(B=-1), dict(P=-1),
               dict(T=1 << 31), dict(q=None), dict(kp=None), dict(v=None), dict(out=None), dict(lengths=None),
               dict(scratch=None), dict(bytes=16), dict(status=None), dict(strides=None), dict(scores=buf), dict(scores_out=buf),
               dict(q=ctypes.c_void_p(4100)), dict(vp=ctypes.c_void_p(4098)), dict(scale=0.0), dict(scale=-1.0),
               dict(scale=float("nan")), dict(strides=[1024, 1024, 132] + [256, 128] * 2 + [2048, 256, 128] * 2),
               dict(strides=[-8] + [1024, 128] + [256, 128] * 2 + [2048, 256, 128] * 2)):
        assert call(**kw) == _lib.ERR_ARG, kw
    assert call(B=0) == _lib.OK and call(Tq=0) == _lib.OK
    assert L.lsa_shared_prefix_scratch(2, 2, 1, 8, 2, 100, 16, 8, 0) == _lib.ERR_ARG
    assert L.lsa_shared_prefix_scratch(2, 2, 1, 8, 2, 128, 16, 8, 1) > 0


def test_evict_entry_refuses_before_any_cuda_call():
    L = _lib_or_skip()
    buf = ctypes.c_void_p(4096)
    ok = dict(k=buf, v=buf, row=256, strides=[4096, 512, 256] * 2, scores=buf, lengths=buf, B=2, T=8, Hkv=2, budget=4,
              window=1, sink=1, capacity=4, ko=buf, vo=buf, so=buf, lo=buf, ids=buf)

    def call(**kw):
        a = dict(ok, **kw)
        st = None if a["strides"] is None else (ctypes.c_int64 * 6)(*a["strides"])
        return L.lsa_evict(a["k"], a["v"], a["row"], st, a["scores"], a["lengths"], a["B"], a["T"], a["Hkv"],
                           a["budget"], a["window"], a["sink"], a["capacity"], a["ko"], a["vo"], a["so"], a["lo"],
                           a["ids"], None)

    for kw in (dict(row=24), dict(row=0), dict(budget=-1), dict(window=4), dict(sink=4), dict(window=-1),
               dict(capacity=3), dict(Hkv=0), dict(T=-1), dict(strides=None), dict(strides=[4096, 512, 8] * 2),
               dict(k=None), dict(scores=None), dict(ids=None), dict(lo=None), dict(lengths=None),
               dict(ko=ctypes.c_void_p(4104))):
        assert call(**kw) == _lib.ERR_ARG, kw
    assert call(B=0) == _lib.OK
