"""Scratch of the shared-prefix attention, without a GPU: a call's parts are bounded by its rows and the
GPU's places, whatever the splits of its last row tiles."""

import random

import pytest

from lsa_b200 import _lib

BF16, F32 = 2, 0
SPLIT = 8 * 148 * 256  # rows of the split tiles' parts, at most


def _scratch(dtype, B, Tq, Hq, Hkv, D, P, T, scored):
    try:
        L = _lib.lib()
    except OSError as e:
        pytest.skip(f"CUDA runtime not loadable here: {e}")
    return L.lsa_shared_prefix_scratch(dtype, B, Tq, Hq, Hkv, D, P, T, scored)


@pytest.mark.parametrize("B,Tq,P", [
    (18, 64, 10007), (19, 64, 10007), (37, 64, 10007), (56, 64, 10007), (500, 64, 10007), (1, 129088, 32768),
    (8, 9664, 32768), (32, 17280, 10007), (1, 64000, 32768),
])
def test_prompt_calls_hold_parts_of_split_tiles_alone(B, Tq, P):
    """Whole tiles write the output themselves: beside four bytes a row there are the split tiles' parts."""
    rows = B * Tq * 32
    assert 0 < _scratch(BF16, B, Tq, 32, 8, 128, P, Tq, 0) <= rows * 4 + SPLIT * 129 * 4 + 1024


@pytest.mark.parametrize("Tq", range(64, 131072, 4032))
def test_one_sequence_of_any_length(Tq):
    assert 0 < _scratch(BF16, 1, Tq, 32, 8, 128, 32768, Tq, 0) <= Tq * 32 * 4 + SPLIT * 129 * 4 + 1024


def test_any_call_is_bounded():
    """Three parts a row (prefix, and a cache's two streams) or the split tiles', for each of the two kinds of
    keys; logits for up to 64 rows a KV head where they are kept."""
    rng = random.Random(1)
    log = lambda low, high: round(low * (high / low) ** rng.random())
    for _ in range(4000):
        Hkv, G, D = log(1, 64), rng.choice([1, 2, 3, 4, 6, 7, 8, 16, 64]), rng.choice([64, 128])
        B, Tq = log(1, 4096), rng.choice([1, 1, 2, 5, log(1, 20000)])
        P, T = rng.choice([0, log(1, 1 << 20)]), rng.choice([0, log(1, 1 << 20)])
        rows = B * Tq * Hkv * G
        if rows > 1 << 30:
            continue
        for dtype in (BF16, F32):
            for scored in (0, 1):
                logits = rows * (T + 15) * 4 if scored and Tq * G <= 64 and dtype == BF16 else 0
                most = 3 * rows * (D + 1) * 4 + 2 * SPLIT * (D + 1) * 4 + rows * 4 + logits + 1024
                got = _scratch(dtype, B, Tq, Hkv * G, Hkv, D, P, T, scored)
                assert 0 < got <= most, (dtype, B, Tq, Hkv * G, Hkv, D, P, T, scored, got / most)
