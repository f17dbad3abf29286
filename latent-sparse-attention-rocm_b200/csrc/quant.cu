// quant.cu - attention over the 8-bit paged cache: the entry points and their plans (sm_100a).
// quant.cuh has the formulas.
#include <math.h>

#include "prefix.cuh"
#include "quant.cuh"

namespace lsa {
namespace {

constexpr int kSMs = 148;
constexpr int kUnit = 128;      // keys that a CTA's four warps take at a time
constexpr int kMaxTileParts = 32, kMostRounds = 8;  // splits of a tile; rounds of the SMs that split tiles fill
constexpr double kItemCost = 1.5, kJoinCost = 3.0;  // a CTA's start and end, the join's launch, in units' times

struct Plan {
    int parts;
    bool cluster;       // joined within clusters of `parts` CTAs
    int tokens, tiles, whole;  // QuantArgs'
    bool streams;
    int64_t part_rows;
    int64_t bytes;      // of scratch
};

// keys: the most that a row sees
Plan make_plan(int64_t B, int64_t Tq, int64_t Hq, int64_t Hkv, int64_t D, int64_t keys, bool lists) {
    Plan p = {};
    const int64_t G = Hq / Hkv, chunks = (keys + kUnit - 1) / kUnit;
    p.part_rows = B * Tq * Hq;
    p.parts = 1;
    // The few-row kernel reads the keys once for each 32 rows, from L2 after the first time, and converts them in
    // registers; the tensor-core kernel's converting goes through shared memory, which its products share, and its start
    // takes 4 us (us, few-row / tensor cores: 32 x 4096 keys, 32 rows 85 / 105, 48 rows 145 / 107; 1 x 65536 32 rows 37 / 45,
    // 64 rows 61 / 44; 4 x 2048 64 rows 20.8 / 20.2; 1 x 2048 128 rows 16.4 / 18.1, 256 rows 20.0 / 24.2; 1 x 512 128 rows
    // 10.6 / 13.4). Many sequences hide that kernel's chains and leave its join's traffic: 48 rows, 64 x 2048 145 / 126,
    // 128 x 2048 236 / 246, 1024 x 1024 1070 / 1373. Lists are the few-row kernel's at any size: the tensor-core kernel reads
    // whole chunks of a sequence and knows none.
    const int64_t rows = Tq * G, heads = B * Hkv * (keys < kUnit ? kUnit : keys);
    const bool few = lists || rows <= 32 || (rows <= 64 && (heads <= 1 << 16 || B * Hkv > 6 * kSMs)) ||
                     (heads <= 1 << 21 && rows * heads <= 1 << 21);
    if (!few && G <= 128) {
        // Whole rounds of one tile an SM are not split (no parts to write, read and join); the tiles of the last, short
        // round are, so that it too fills the GPU.
        p.tokens = (int)(128 / G);
        p.tiles = (int)((Tq + 2 * p.tokens - 1) / (2 * p.tokens));
        const int64_t all = B * Hkv * p.tiles;
        // Two streams write two parts a row: of more items than kMostRounds they would want more scratch than the other
        // calls and gain nothing by it (96 rows, streams / whole tiles: 128 x 2048 261 / 292, 256 x 2048 507 / 572, 512 x
        // 1024 707 / 687, 1024 x 512 1142 / 956).
        p.streams = Tq <= p.tokens && all <= kMostRounds * kSMs;
        const int64_t split = p.streams ? all : all % kSMs;
        const int64_t most = split ? kMostRounds * kSMs / split : 0;
        p.parts = balance(split, chunks, 4, kSMs, (int)(most < 1 ? 1 : (most < kMaxTileParts ? most : kMaxTileParts)));
        if (p.parts < 1) p.parts = 1;
        // two streams are parts of their own: they never write the output
        p.whole = (int)(p.streams ? 0 : (p.parts == 1 ? all : all - split));
        p.part_rows = (all - p.whole) * quant_tile_rows(p.streams);
        p.bytes = p.part_rows * (p.streams ? 2 : 1) * p.parts * (D + 1) * 4;
        return p;
    }
    const int64_t items = B * Hkv * few_row_tiles(rows, lists);
    // Parts. One CTA in each of two places an SM draws the memory's whole rate; a third place only evens out ragged
    // sequences, and a round that fills some SMs' third place and not others' is the worst (us in parts, CTAs in
    // brackets; 32 / 8 heads, D 128): 1 x 32k 37 (296) 16.1, 42 (336) 17.8, 56 (448) 20.2; 4 x 16k 9 (288) 24.5, 14 (448)
    // 29.5; 16 x 8k 2 (256) 41.9, 3 (384) 39.3, 5 (640) 44.1; 32 x 4k 1 (256) 49.0, 3 (768) 40.9; 64 x 8k 1 (512) 156,
    // 4 (2048) 133, 12 (6144) 155. Lists are of one length: rounds of two places.
    int64_t s;
    if (lists) {
        s = balance(items, chunks, kItemCost, 2 * kSMs, kMaxQuantParts);
        auto cost = [&](int64_t n) {
            return (double)((items * n + 2 * kSMs - 1) / (2 * kSMs)) * ((double)chunks / n + kItemCost);
        };
        if (s > 1 && cost(s) + kJoinCost >= cost(1)) s = 1;
    } else if (items <= 100) {
        s = 2 * kSMs / items;
    } else if (items <= 200) {
        s = (2 * kSMs + kSMs * 2 / 3) / items;
    } else {
        s = 2048 / items < chunks / 8 ? 2048 / items : chunks / 8;
    }
    if (s > chunks) s = chunks;
    if (s > kMaxQuantParts) s = kMaxQuantParts;
    p.parts = s < 1 ? 1 : (int)s;
    // Parts that are a cluster's CTAs join within the launch, which pays where a CTA has little to do (4 x 2k keys, 8
    // parts: 7.2 us against 10.5); clusters spread unevenly over the SMs (4 x 16k, 8 parts: 29.4 us, in a second launch
    // 25.3).
    int c = 1;
    while (2 * c <= kMostCluster && 2 * c <= s && (c < 8 || items * 2 * c <= kSMs)) c *= 2;
    if (c > 1 && (chunks <= 3 * c || (items * c <= kSMs && chunks <= 4 * c))) p.parts = c, p.cluster = true;
    p.bytes = p.parts > 1 && !p.cluster ? p.parts * p.part_rows * (D + 1) * 4 : 0;
    return p;
}

bool sizes_ok(int64_t B, int64_t Tq, int64_t Hq, int64_t Hkv, int64_t D, int64_t keys) {
    if (B < 0 || Tq < 0 || keys < 0 || Hkv < 1 || Hq < 1 || Hq % Hkv != 0 || (D != 64 && D != 128)) return false;
    if (B > 65535 || Tq > (1 << 24) || Hq > 65536 || keys > (1 << 30)) return false;
    if (Tq * (Hq / Hkv) > (1 << 30) || Tq * (Hq / Hkv) * (Hq / Hkv) > UINT32_MAX) return false;  // token_of
    return B * Tq <= (int64_t)INT32_MAX / Hq;
}

int pool(QuantArgs* a, const void* k8, const void* v8, const float* ks, const float* vs, int code, int64_t pages,
         int64_t page, int64_t Hkv, const int32_t* table, int64_t table_ld, int64_t table_rows, int64_t M,
         const int32_t* lengths) {
    if (code != kE4M3 && code != kInt8) return LSA_ERR_ARG;
    if (page != 16 && page != 32 && page != 64 && page != 128) return LSA_ERR_ARG;
    if (pages < 0 || M < 0 || table_ld < 0 || table_rows < 0) return LSA_ERR_ARG;
    if (M > (1 << 30) / page || pages > INT32_MAX / (page * Hkv) || table_rows > INT32_MAX) return LSA_ERR_SIZE;
    if (lengths == nullptr || (M > 0 && table == nullptr)) return LSA_ERR_ARG;
    if (pages > 0 && (!k8 || !v8 || !ks || !vs)) return LSA_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(k8) % 16 != 0 || reinterpret_cast<uintptr_t>(v8) % 16 != 0) return LSA_ERR_ARG;
    a->k8 = static_cast<const uint8_t*>(k8), a->v8 = static_cast<const uint8_t*>(v8);
    a->ks = ks, a->vs = vs;
    a->table = table, a->table_ld = table_ld, a->table_rows = (int)table_rows, a->pages = (int)pages;
    a->M = pages > 0 ? (int)M : 0;  // an empty pool holds nothing
    a->shift = page == 16 ? 4 : (page == 32 ? 5 : (page == 64 ? 6 : 7));
    a->lengths = lengths;
    return LSA_OK;
}

int run(QuantArgs& a, int dtype, int code, int64_t D, int64_t keys, float scale, void* scratch, int64_t scratch_bytes,
        cudaStream_t stream) {
    a.scale_log2 = scale * 1.4426950408889634f;
    if (!(a.scale_log2 > 0) || !isfinite(a.scale_log2)) return LSA_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(a.q) % 16 != 0 || reinterpret_cast<uintptr_t>(a.out) % 16 != 0) return LSA_ERR_ARG;
    for (int64_t st : {a.q_b, a.q_t, a.q_h})
        if (st < 0 || st % 8 != 0) return LSA_ERR_ARG;
    a.G_inverse = a.G > 1 ? (uint32_t)(((1ull << 32) + a.G - 1) / a.G) : 0;
    const Plan p = make_plan(a.B, a.Tq, a.Hq, a.Hkv, D, keys, a.lists != nullptr);
    if (p.bytes > 0 && (scratch == nullptr || scratch_bytes < p.bytes || reinterpret_cast<uintptr_t>(scratch) % 16 != 0))
        return LSA_ERR_ARG;
    a.rows = (int64_t)a.B * a.Tq * a.Hq;
    a.parts = p.parts, a.cluster = p.cluster;
    a.tokens = p.tokens, a.tiles = p.tiles, a.whole = p.whole, a.streams = p.streams;
    a.part_rows = p.part_rows;
    a.wait_ns = wait_limit_ns();
    a.part_o = static_cast<float*>(scratch);
    a.part_lse = a.part_o + (p.streams ? 2 : 1) * p.parts * p.part_rows * D;
    const int rc = a.tokens > 0 ? launch_quant_tiles(a, dtype, code, (int)D, stream)
                                : launch_quant_rows(a, dtype, code, (int)D, stream);
    return rc != LSA_OK || p.bytes == 0 ? rc : launch_quant_join(a, dtype, (int)D, stream);
}

}  // namespace
}  // namespace lsa

extern "C" {

int64_t lsa_quantized_scratch(int64_t B, int64_t Tq, int64_t Hq, int64_t Hkv, int64_t D, int64_t keys, int lists) {
    using namespace lsa;
    if (!sizes_ok(B, Tq, Hq, Hkv, D, keys)) return LSA_ERR_ARG;
    if (B == 0 || Tq == 0) return 0;
    const Plan p = make_plan(B, Tq, Hq, Hkv, D, keys, lists != 0);
    if (p.tokens == 0 && Hkv * few_row_tiles(Tq * (Hq / Hkv), lists != 0) > 65535) return LSA_ERR_SIZE;
    return p.bytes;
}

int lsa_quantized_attention(const void* q, int dtype, const int64_t* q_strides, const void* k8, const void* v8,
                            const float* k_scale, const float* v_scale, int code, int64_t pages, int64_t page,
                            const int32_t* table, int64_t table_ld, int64_t M, const int32_t* lengths, int64_t B,
                            int64_t Tq, int64_t Hq, int64_t Hkv, int64_t D, float scale, void* out, float* lse,
                            void* scratch, int64_t scratch_bytes, int32_t* status, cudaStream_t stream) {
    using namespace lsa;
    if (page < 16 || page > 128 || M < 0 || M > (1 << 30)) return LSA_ERR_ARG;
    if ((dtype != kF16 && dtype != kBF16) || !sizes_ok(B, Tq, Hq, Hkv, D, M * page)) return LSA_ERR_ARG;
    if (B == 0 || Tq == 0) return LSA_OK;
    if (q == nullptr || out == nullptr || q_strides == nullptr || status == nullptr) return LSA_ERR_ARG;
    QuantArgs a = {};
    const int rc = pool(&a, k8, v8, k_scale, v_scale, code, pages, page, Hkv, table, table_ld, B, M, lengths);
    if (rc != LSA_OK) return rc;
    a.q = q, a.q_b = q_strides[0], a.q_t = q_strides[1], a.q_h = q_strides[2];
    a.out = out, a.lse = lse, a.status = status;
    a.B = (int)B, a.Tq = (int)Tq, a.Hq = (int)Hq, a.Hkv = (int)Hkv, a.G = (int)(Hq / Hkv);
    return run(a, dtype, code, D, M * page, scale, scratch, scratch_bytes, stream);
}

int lsa_quantized_read(const void* q, int dtype, const int64_t* q_strides, const void* k8, const void* v8,
                       const float* k_scale, const float* v_scale, int code, int64_t pages, int64_t page,
                       const int32_t* table, int64_t table_ld, int64_t table_rows, int64_t M, const int32_t* lengths,
                       const int32_t* lists, const int32_t* counts, const int32_t* rows, int64_t R, int64_t W,
                       int64_t Hq, int64_t Hkv, int64_t D, float scale, void* out, void* scratch,
                       int64_t scratch_bytes, cudaStream_t stream) {
    using namespace lsa;
    if ((dtype != kF16 && dtype != kBF16) || !sizes_ok(R, 1, Hq, Hkv, D, W)) return LSA_ERR_ARG;
    if (R == 0) return LSA_OK;
    if (q == nullptr || out == nullptr || q_strides == nullptr || counts == nullptr || (W > 0 && lists == nullptr))
        return LSA_ERR_ARG;
    if (rows == nullptr && table_rows < R) return LSA_ERR_ARG;
    QuantArgs a = {};
    const int rc = pool(&a, k8, v8, k_scale, v_scale, code, pages, page, Hkv, table, table_ld, table_rows, M, lengths);
    if (rc != LSA_OK) return rc;
    a.q = q, a.q_b = q_strides[0], a.q_t = 0, a.q_h = q_strides[1];
    a.lists = W > 0 ? lists : counts;  // without entries nothing is read of it
    a.counts = counts, a.list_rows = rows, a.W = a.M > 0 ? (int)W : 0;
    a.out = out, a.lse = nullptr;
    a.B = (int)R, a.Tq = 1, a.Hq = (int)Hq, a.Hkv = (int)Hkv, a.G = (int)(Hq / Hkv);
    return run(a, dtype, code, D, W, scale, scratch, scratch_bytes, stream);
}

}  // extern "C"
