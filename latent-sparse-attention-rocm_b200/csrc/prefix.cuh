// prefix.cuh - what the kernels of the shared-prefix attention share (sm_100a).
//
// B sequences read the same P prefix keys, stored once, and then their own caches. Query row
// (b, i) of Tq sees every prefix key and the own keys j < lengths[b] - Tq + i + 1 (lengths
// count the call's Tq new tokens). For a (query row, query head) pair with logits
// s_j = scale (q . k_j):
//   m = max s_j,  l = sum e^(s_j - m),  o = sum e^(s_j - m) v_j / l,  lse = m + log l.
// Sums over disjoint key ranges ("parts": the prefix's splits, the own cache's splits) join by
//   o = sum_c 2^(lse_c - M) o_c / sum_c 2^(lse_c - M),  M = max lse_c
// (lse in the log2 domain), so the prefix is one product of all sequences' rows with keys that
// are read once, whatever the batch. A pair that sees no key reads as zeros, lse -inf.
#pragma once

#include <stdint.h>

#include "launch.cuh"

namespace lsa {

constexpr int kMaxSplits = 32;  // of the prefix, and of the own caches (few rows: three times that)
constexpr int kMaxParts = 256;  // of a row: at most 96 + 96, or 64 + 64 (two parts a split), or 96 + 64

// strides in elements; the last dimension is contiguous everywhere
struct PrefixArgs {
    const void *q, *kp, *vp, *k, *v;
    int64_t q_b, q_t, q_h;                // q [B, Tq, Hq, D]
    int64_t kp_t, kp_h, vp_t, vp_h;       // prefix [P, Hkv, D]
    int64_t k_b, k_t, k_h, v_b, v_t, v_h; // own [B, T, Hkv, D]
    const int32_t* lengths;               // [B]
    void* out;                            // [B, Tq, Hq, D] contiguous
    float* part_o;                        // [parts][part_rows][D], each part normalised by its own sum
    float* part_lse;                      // [parts][part_rows], log2 domain, -inf: no key
    float* lse2;                          // [rows], log2 domain: the joined lse
    float* lse;                           // [rows], natural, or null
    int B, Tq, Hq, Hkv, G;
    int P, T;
    int Sp, So;                           // splits of the prefix and of the own caches
    int parts_p, parts_o;                 // parts of a row from the prefix and from its own cache
    int64_t rows;                         // B * Tq * Hq
    int64_t part_rows;                    // rows, or 256 a split tile where whole tiles have no parts (TilePlan::whole)
    float scale_log2;                     // scale * log2(e)
    int32_t* status;                      // LSA_ERR_TIMEOUT after an expired wait
    uint64_t wait_ns;                     // limit of each wait of the tensor-core kernels
};

// The work of the tensor-core kernel (prefix_tile.cu). A row tile is two halves of `tokens` tokens,
// the G query heads of each (at most 128 rows a half).
struct TilePlan {
    int tokens;                    // 128 / G

    int batch_items, batch_tiles;  // row tiles over all sequences: prefix keys
    int seq_items, seq_tiles;      // row tiles of a sequence: its own keys (items; tiles of a sequence)
    bool batch_streams, seq_streams;  // tiles of one half's rows: two streams of chunks
    bool joint;                    // seq tiles read the prefix too
    int whole;                     // the first seq tiles, not split: they write the output themselves
};

// Row rl of half `hf` of a row tile: (token of the tile, head of the group); false: no row there.
__device__ __forceinline__ bool tile_row(const PrefixArgs& a, const TilePlan& t, int hf, int rl, int* tok, int* g) {
    const int tl = rl / a.G;
    *tok = hf * t.tokens + tl;
    *g = rl - tl * a.G;
    return tl < t.tokens;
}

// Seq tile i: (sequence, KV head, row tile), the longest causal ranges first.
__device__ __forceinline__ void seq_tile(const PrefixArgs& a, const TilePlan& t, int i, int* b, int* h, int* tile) {
    *h = i % a.Hkv, i /= a.Hkv;
    *b = i % a.B;
    *tile = t.seq_tiles - 1 - i / a.B;
}

// Splits of `chunks` for `items` equal work items on `slots` places that hold one item each: the
// fewest that minimise rounds x (chunks of an item + its fixed cost in chunks).
inline int balance(int64_t items, int64_t chunks, double fixed, int64_t slots, int most) {
    if (chunks == 0) return 0;
    int best = 1;
    double least = 1e300;
    for (int s = 1; s <= most && s <= chunks; ++s) {
        const double cost = (double)((items * s + slots - 1) / slots) * ((double)chunks / s + fixed);
        if (cost < 0.99 * least) least = cost, best = s;
    }
    return best;
}

// The same for work that shares the GPU with `beside` chunks' worth of other work per place, which
// starts on the places left free: the least of the longer of its own rounds and all the work together.
inline int balance_beside(int64_t items, int64_t chunks, double fixed, int64_t slots, double beside, int most) {
    if (chunks == 0) return 0;
    int best = 1;
    double least = 1e300;
    for (int s = 1; s <= most && s <= chunks; ++s) {
        const double one = (double)chunks / s + fixed;
        const double alone = (double)((items * s + slots - 1) / slots) * one;
        const double all = (double)(items * s) * one / slots + beside;
        const double cost = alone > all ? alone : all;
        if (cost < 0.99 * least) least = cost, best = s;
    }
    return best;
}

// own keys that sequence b holds
__device__ __forceinline__ int own_length(const PrefixArgs& a, int b) {
    const int n = a.lengths[b];
    return n < 0 ? 0 : (n > a.T ? a.T : n);
}

// row r of KV head h in a segment's row order ((token, query head of the group) pairs):
// the row's place in q / out and its index among all rows
__device__ __forceinline__ int64_t row_index(const PrefixArgs& a, int64_t token, int h, int g) {
    return token * a.Hq + (int64_t)h * a.G + g;
}

// The part of [0, n) that split s of S takes, in units of `unit` keys: sizes differ by one unit.
__device__ __host__ __forceinline__ void split_range(int n, int s, int S, int unit, int* k0, int* k1) {
    const int64_t units = ((int64_t)n + unit - 1) / unit;
    const int64_t a = units * s / S * unit, b = units * (s + 1) / S * unit;
    *k0 = (int)(a < n ? a : n);
    *k1 = (int)(b < n ? b : n);
}

// The work of the few-row kernel (prefix_rows.cu), 16 rows of a KV head an item.
struct RowsPlan {
    int prefix_items, own_items;
    int own_tiles;  // row tiles of a sequence (the prefix's rows are one tile)
    bool follows;   // launched behind this call's tensor-core kernel, whose output it does not read
    int64_t pitch;  // T to whole tiles of 16 keys
    float* logits;  // [B, Hkv, Tq * G, pitch] log2-domain logits of the own keys, or null
};

// The limit of each bounded wait of the calls launched from now on (lsa_shared_prefix_wait_limit).
uint64_t wait_limit_ns();

int launch_prefix_simt(const PrefixArgs& a, int D, cudaStream_t stream);  // fp32 inputs
int launch_prefix_tiles(const PrefixArgs& a, const TilePlan& tp, int dtype, int D, cudaStream_t stream);
int launch_prefix_rows(const PrefixArgs& a, const RowsPlan& rp, int dtype, int D, cudaStream_t stream);
// The parts joined; with logits (few-row kernel) also the own keys' weights, in the same launch.
int launch_prefix_finish(const PrefixArgs& a, const TilePlan& tp, int dtype, int D, const RowsPlan& rp,
                         const float* scores, float* scores_out, cudaStream_t stream);
int launch_own_weights(const PrefixArgs& a, int D, const float* scores, float* scores_out, cudaStream_t stream);
int launch_tile_weights(const PrefixArgs& a, int dtype, int D, const float* scores, float* scores_out,
                        cudaStream_t stream);

}  // namespace lsa
