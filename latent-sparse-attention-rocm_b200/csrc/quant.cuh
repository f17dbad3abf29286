// quant.cuh - what the kernels of the 8-bit paged cache share (sm_100a).
//
// A pool holds pages of `page` tokens (16, 32, 64 or 128): codes [pages, Hkv, page, D] of K and of V, e4m3 or
// 8-bit integers, and one fp32 scale a (page, KV head) of each. Token t of sequence b is row t % page of page
// table[b][t / page]; its key is ks * code. A (page, head)'s rows are contiguous (page x D bytes), so a tile of
// keys is whole 128-byte lines whatever the page order.
//
// For a query row with logits s_j = scale ks_j (q . k8_j) (log2 domain below) the value scale goes into the
// exponent: t_j = s_j + log2 vs_j, m = max t_j, P_j = 2^(t_j - m), l = sum P_j / vs_j,
//   o = sum P_j v8_j / l,   lse = m + log2 l.
// One exponential a key serves both sums, P_j is at most 1 whatever the scales, and the values' codes enter
// their product as they are. Exact as long as a sequence's value scales lie within 2^100 of each other
// (beyond, a P_j may be lost to underflow that l should see): they count as at least 2^-60, the floor of the
// append's scales.
#pragma once

#include <cuda_fp8.h>

#include <type_traits>

#include "launch.cuh"

namespace lsa {

enum Code : int { kE4M3 = 0, kInt8 = 1 };

constexpr int kMinExponent = -60;  // of a scale that the append writes
constexpr int kMaxQuantParts = 96;
constexpr int kMostCluster = 16;

struct QuantArgs {
    const void* q;
    int64_t q_b, q_t, q_h;        // strides of q [B, Tq, Hq, D], in elements
    const uint8_t *k8, *v8;       // [pages, Hkv, page, D]
    const float *ks, *vs;         // [pages, Hkv]
    const int32_t* table;         // [table_rows, M], rows table_ld apart
    int64_t table_ld;
    int table_rows, M, pages, shift;  // page = 1 << shift
    const int32_t* lengths;       // [table_rows]
    const int32_t *lists, *counts, *list_rows;  // read: [B, W] positions, [B], [B]
    int W;
    void* out;                    // [B, Tq, Hq, D] contiguous
    float *part_o, *part_lse;     // [parts][rows][D] (normalised), [parts][rows] (log2 domain; -inf: no key)
    float* lse;                   // [rows] natural, or null
    int B, Tq, Hq, Hkv, G;
    uint32_t G_inverse;           // ceil(2^32 / G); 0 for G = 1
    int parts;
    bool cluster;                 // the parts are a cluster's CTAs, which join them (few-row kernel)
    int64_t rows;                 // B * Tq * Hq
    // The tensor-core kernel's (quant_tile.cu): tokens of a half tile (0: the few-row kernel), tiles of a sequence and
    // KV head, whether a tile is one half's rows, and the first tiles, which are not split and write the output
    // themselves. A part then has the split tiles' rows, quant_tile_rows(a) a tile.
    int tokens, tiles, whole;
    bool streams;
    int64_t part_rows;            // rows of a part
    int32_t* status;              // LSA_ERR_TIMEOUT after an expired wait
    uint64_t wait_ns;             // limit of each wait
    float scale_log2;             // scale * log2(e)
};

// Two codes, bytes 2 hi and 2 hi + 1 of a word, as a pair of halves (exact: e4m3's values and whole numbers up
// to 128 are halves).
template <int CODE> __device__ __forceinline__ uint32_t halves_of(uint32_t word, int hi);
template <> __device__ __forceinline__ uint32_t halves_of<kE4M3>(uint32_t word, int hi) {
    uint32_t r;
    if (hi)
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, b;\n\t}" : "=r"(r) : "r"(word));
    else
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t}" : "=r"(r) : "r"(word));
    return r;
}
template <> __device__ __forceinline__ uint32_t halves_of<kInt8>(uint32_t word, int hi) {
    // byte + 128 in the low bits of 1024's mantissa, then 1152 off
    const uint32_t u = __byte_perm(word ^ 0x80808080u, 0x64646464u, hi ? 0x4342 : 0x4140);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Four fp32 values -> four codes, to the nearest (ties to even).
template <int CODE> __device__ __forceinline__ uint32_t codes_of(float a, float b, float c, float d);
template <> __device__ __forceinline__ uint32_t codes_of<kE4M3>(float a, float b, float c, float d) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
        "mov.b32 %0, {l, h};\n\t}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
}
template <> __device__ __forceinline__ uint32_t codes_of<kInt8>(float a, float b, float c, float d) {
    auto one = [](float x) { return (uint32_t)min(127, max(-127, __float2int_rn(x))) & 0xFFu; };
    return one(a) | one(b) << 8 | one(c) << 16 | one(d) << 24;
}

// The smallest power of two s >= 2^kMinExponent with top <= (the code's largest value) * s, as bits.
template <int CODE> __device__ __forceinline__ float scale_for(float top) {
    const uint32_t bits = __float_as_uint(top);
    // 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
    const uint32_t last = CODE == kE4M3 ? 0x600000u : 0x7E0000u;
    int e = (int)(bits >> 23) - 127 - (CODE == kE4M3 ? 8 : 6) + ((bits & 0x7FFFFFu) > last ? 1 : 0);
    e = e < kMinExponent ? kMinExponent : e;
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// The power of two that brings a bf16 row to fp16, its largest magnitude (bits given) to [2^8, 2^9); *factor takes its
// inverse. Zero, infinities and NaN stay as they are.
__device__ __forceinline__ float half_factor(uint32_t top, float* factor) {
    const int e = (int)(top >> 7);  // biased exponent
    const int up = e == 0 || e == 255 ? 0 : min(8 - (e - 127), 100);
    *factor *= __uint_as_float((uint32_t)(127 - up) << 23);
    return __uint_as_float((uint32_t)(up + 127) << 23);
}

// A row of q that is not finite (its largest magnitude's bits say) enters the products as zeros, with a factor of -0, so that
// it is NaN only where a key is seen: a key that is not there has zeros for its codes, and NaN times those would make
// rows without keys NaN. At the end its sum becomes NaN unless it is 0. (A finite row's factor is never -0. A row with
// an infinity has only infinities and NaN for logits, so NaN is its softmax over any keys.)
template <typename T> __device__ __forceinline__ bool infinite_row(uint32_t top) {
    return top >= (std::is_same<T, __nv_bfloat16>::value ? 0x7F80u : 0x7C00u);
}
constexpr float kInfiniteRow = -0.0f;
__device__ __forceinline__ float sum_of_row(float sum, float factor) {
    return __float_as_uint(factor) == 0x80000000u && sum != 0.0f ? __uint_as_float(0x7FFFFFFFu) : sum;
}

// Token of row r of a (sequence, KV head), r < Tq G: r / G, exact for r G below 2^32 (the entry point checks).
__device__ __forceinline__ int token_of(const QuantArgs& a, int r) {
    return a.G_inverse ? (int)__umulhi((uint32_t)r, a.G_inverse) : r;
}

// Tile i of the tensor-core kernel: (sequence, KV head, row tile), the longest causal ranges first.
__device__ __forceinline__ void quant_tile_at(const QuantArgs& a, int i, int* b, int* h, int* tile) {
    *h = i % a.Hkv, i /= a.Hkv;
    *b = i % a.B;
    *tile = a.tiles - 1 - i / a.B;
}
__host__ __device__ __forceinline__ int quant_tile_rows(bool streams) { return streams ? 128 : 256; }
// Row rl of half hf of split tile `rest`, in part `split` (two parts a split where the halves are streams).
__device__ __forceinline__ int64_t quant_part_row(const QuantArgs& a, int split, int rest, int hf, int rl) {
    return a.streams ? (2 * split + hf) * a.part_rows + (int64_t)rest * 128 + rl
                     : split * a.part_rows + (int64_t)rest * 256 + hf * 128 + rl;
}

// Rows of the few-row kernel's tiles for so many rows of a sequence and KV head.
inline int few_tile_rows(int64_t rows, bool lists) { return rows <= 16 || lists ? 16 : 32; }
inline int64_t few_row_tiles(int64_t rows, bool lists) {
    return (rows + few_tile_rows(rows, lists) - 1) / few_tile_rows(rows, lists);
}

int launch_quant_tiles(const QuantArgs& a, int dtype, int code, int D, cudaStream_t stream);
int launch_quant_rows(const QuantArgs& a, int dtype, int code, int D, cudaStream_t stream);
int launch_quant_join(const QuantArgs& a, int dtype, int D, cudaStream_t stream);

}  // namespace lsa
