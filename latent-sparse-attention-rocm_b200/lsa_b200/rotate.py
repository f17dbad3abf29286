"""Norms of queries and keys for each head, with the position rotation, in one pass.

What a model does between its projections and everything this package starts from: the index
space (``make_index_space``), the caches and every read take q and k as these leave them. No
reference counterpart: the reference is handed rotated queries and keys.

    f, amplitude = rotary_frequencies(128, base=500000.0, scaling="yarn", factor=8.0, trained=16384)
    q, k = norm_rotate(q, k, positions, f.cuda(), q_norm, k_norm, amplitude=amplitude)
"""

from __future__ import annotations

import math

import torch

from . import _lib


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       trained: int = 0, fast: float = 32.0, slow: float = 1.0):
    """(frequencies, amplitude): radians a position of the ``dim / 2`` pairs, fp64 on the CPU, and
    the factor of the rotated values.

    ``base ** (-2 i / dim)``, for long contexts scaled by one of: "linear", every frequency over
    ``factor`` (position interpolation); "ntk", the base raised so that the slowest pair alone is
    slowed by ``factor``; "yarn", pairs that turn more than ``fast`` times within ``trained``
    positions as they are, those below ``slow`` turns over ``factor``, a ramp between, and the
    amplitude ``0.1 ln(factor) + 1``."""
    if dim < 2 or dim % 2:
        raise ValueError(f"rotary_frequencies: an even number of dimensions, got {dim}")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"rotary_frequencies: scaling none, linear, ntk or yarn, got {scaling!r}")
    if not (base > 1 and factor >= 1 and math.isfinite(base) and math.isfinite(factor)):
        raise ValueError(f"rotary_frequencies: base above 1 and factor at least 1, got {base}, {factor}")
    i = torch.arange(dim // 2, dtype=torch.float64)
    if scaling == "ntk" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    f = base ** (-2.0 * i / dim)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling != "yarn":
        return f, 1.0
    if trained < 1 or not fast > slow > 0:
        raise ValueError("rotary_frequencies: yarn takes the trained length, and fast above slow above 0")

    def pair(turns):  # the (real) index of the pair that turns so often within the trained length
        return dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dim - 1)
    ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
    if pair(slow) < 0:  # the first pair turns less often too: the ramp ends before it
        ramp = torch.ones_like(i)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0


def norm_rotate(q, k, positions, frequencies, q_weight=None, k_weight=None, eps: float = 1e-6,
                interleaved: bool = False, amplitude: float = 1.0):
    """(q, k): every head's root-mean-square norm, where a weight is given, and the rotation.

    q [B, T, Hq, D], k [B, T, Hkv, D] (fp32, fp16 or bf16; D 64, 128 or 256; strided views such as slices of
    a joint projection as they are, the head dimension contiguous and rows on 16-byte boundaries);
    ``positions`` [B, T], or [T] for all sequences, whole numbers, negative ones too. The weights [D]
    have q's type or fp32; without one its tensor is not normalised. ``frequencies`` [R / 2] fp64,
    radians a position: the first R values of a head turn (R a multiple of 16, at most D; 0: none),
    value i with value i + R / 2, or 2 i with 2 i + 1 where ``interleaved``, times ``amplitude``; the others
    pass. In fp32 (the squares' sum too: values below 2^60), the angles reduced in fp64, rounded once.
    Outputs contiguous, like q and k."""
    out = _lib.torch_ops().norm_rotate(q, k, positions, frequencies, q_weight, k_weight, eps, interleaved, amplitude)
    _lib.after_call(q.device, "norm_rotate")
    return out
