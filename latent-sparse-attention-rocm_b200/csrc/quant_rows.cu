// quant_rows.cu - attention over the 8-bit paged cache for few rows, and its sparse read (sm_100a).
// quant.cuh has the formulas.
//
// A work item is at most 32 query rows of one KV head (a sequence's last tokens; of the read one token's G query
// heads) x a range of keys. The keys' bytes bound it: 2 D a key and head. So nothing waits for a neighbour in the
// main loop: each of a CTA's four warps copies its own tiles of 32 keys (cp.async, 16 bytes, kRing tiles in
// flight) and runs its own online softmax on them. S^T = K Q^T and O^T += V^T P^T by mma.sync.m16n8k16 in fp16:
// keys, then columns of V, are the M = 16 side and the rows the N = 8 (twice for more than eight, four times for more
// than 16), so few rows cost few accumulators. The codes become halves in registers on their way into the fragments, which is exact:
//   K: a lane takes 16 bytes of key g = lane / 4 at a time, four consecutive bytes a k-step; Q's fragments are
//      loaded in the same order of D, which a product does not see.
//   V: a lane takes D / 8 bytes of four keys and makes pairs of two keys' codes (the fragment's order) by byte
//      permutes; M's rows g and g + 8 are then columns (D / 8) g + 2 j and + 1, put back at the end.
//   P: 8 x 8 blocks transposed by movmatrix.
// Q is made fp16 as well: bf16 rows by an exact power of two that brings their largest value to [2^8, 2^9)
// (what is 2^-22 of it or less loses bits, 2^-33 of it at most), back in the row's factor.
// P is rounded to fp16 for its product. It carries 2^kLift, and the maximum is let stand until it has grown by
// more than 2^kGrow, so P is at most 2^15 and 2^-35 of a row's largest is kept. Sums, maxima and joins are fp32.
//
// Measured (B200, 32 / 8 heads, D 128, bf16, pages of 64, called in a loop, joins included): 64 ragged sequences of up
// to 8191 keys, 807 MB, 133-142 us = 5.7-6.1 TB/s, 88-94 % of the measured copy rate; one of 131072 (int8), 269 MB, 47-52 us;
// 4 of up to 2048 7.2 us as graph replays (a chain of latencies: lengths, pages, two tiles of 1600 cycles, the warps' and
// the cluster's joins), 8.7 to 10 called (the host). 32 rows on 65536 keys 37 us. 32 lists of 2116 keys, 141 MB, 42-45 us:
// rows of 128 bytes all over the pool come at 4.4 TB/s at most (measured with plain loads), and two scale sectors a key
// come with them. A list's rows are fetched again, from L2, for every 16 heads of its group (graph replays: 64 lists, one KV
// head, 64 heads 40 us, 71 heads 65; 8 lists, 128 heads 16). Rows on the M side and keys on the N side
// (an M = 16 tile for four rows) took 183 us for the 64 sequences, its P and O twice as large.
// Not kept: rows of a list asked of L2 ahead (55 us against 44), pages looked up two tiles ahead and the scales'
// logarithms behind S (no change).
#include <type_traits>

#include "prefix_umma.cuh"
#include "quant.cuh"

namespace lsa {
namespace {

constexpr int kWarps = 4;
constexpr int kKeys = 32;  // keys of a warp's tile: one a lane where they are looked up
constexpr int kFewParts = 8;  // that one warp joins
constexpr float kLift = 10.0f, kGrow = 5.0f;

template <int D, int NT, bool LISTS> struct QuantShape {
    static constexpr int kRows = 8 * NT;
    static constexpr int kCTAs = NT == 1 && !LISTS ? 3 : 2;             // an SM
    // tiles in a warp's ring
    static constexpr int kRing = D == 128 ? (kCTAs == 3 || NT == 4 ? 2 : 3) : (kCTAs == 3 || NT == 4 ? 4 : 5);
    static constexpr int kTile = kKeys * D;            // K or V bytes of a tile
    static constexpr int kStage = 2 * kTile + kKeys * 12;  // + ks, vs (then its logarithm) and 1 / vs of every key
    static constexpr int kWarpBytes = (kRing * kStage + 127) / 128 * 128;
    static constexpr int kIn = kWarps * kWarpBytes + kWarps * kRows * 2 * 4;  // what a cluster's CTAs send: sums, lse
    static constexpr int kItems = kRows * D / 4;                              // of 4 columns
    static constexpr int kQ = kIn + kItems * 20;  // Q's fragments and the rows' factors, of 32 rows
    static constexpr int kSmem = kQ + (NT == 4 ? kRows * D * 2 + kRows * 4 : 0);
    static_assert(kWarpBytes >= kRows * D * 4, "the join reuses a warp's ring");
    static_assert(kStage % 16 == 0, "16-byte copies");
};

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, uint32_t src_bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t r;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r) : "r"(addr) : "memory");
    return r;
}
__device__ __forceinline__ uint64_t lds64(uint32_t addr) {
    uint64_t r;
    asm volatile("ld.shared.b64 %0, [%1];" : "=l"(r) : "r"(addr) : "memory");
    return r;
}
// The cluster's barrier, by whole warps.
__device__ __forceinline__ void cluster_arrive() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// The address that CTA `rank` of the cluster has for what this CTA has at `addr`.
__device__ __forceinline__ uint32_t peer(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void send_f4(uint32_t addr, const float4& x) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(x.x), "f"(x.y), "f"(x.z), "f"(x.w)
                 : "memory");
}
__device__ __forceinline__ void send_f1(uint32_t addr, float x) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(x) : "memory");
}
template <typename T> __device__ __forceinline__ void store4(T* dst, const float4& x) {
    const T y[4] = {from_f32<T>(x.x), from_f32<T>(x.y), from_f32<T>(x.z), from_f32<T>(x.w)};
    *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(y);
}
// Block of 8 x 8 halves, lane (g, c) holding [g][2c], [g][2c + 1], transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ void cp_async16_all(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void sts_f32(uint32_t addr, float x) {
    asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(x) : "memory");
}
__device__ __forceinline__ float lg2_approx(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <int N> __device__ __forceinline__ void lds_words(uint32_t (&r)[N], uint32_t addr) {
    if constexpr (N == 4)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(addr)
                     : "memory");
    else
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
}

// Where 16-byte chunk c of key row r of a tile lies: 128-byte lines (two rows each for D = 64). V's chunks are
// permuted so that four keys' rows two apart, read by one instruction, fall into different banks; K's so that two
// neighbours' do.
template <int D> __device__ __forceinline__ uint32_t k_at(int r, int c) {
    return D == 128 ? r * 128 + ((c ^ ((r & 1) << 2)) << 4) : r * 64 + (c << 4);
}
template <int D> __device__ __forceinline__ uint32_t v_at(int r, int c) {
    return D == 128 ? r * 128 + ((c ^ (r & 6)) << 4) : (r >> 1) * 128 + (((((r & 1) << 2) | c) ^ (r & 6)) << 4);
}

// NT: tiles of eight rows. Of four, each warp makes the fragments of one, and they are read from shared memory.
template <typename T, int CODE, int D, bool LISTS, int NT>
__global__ void __launch_bounds__(kWarps * 32, QuantShape<D, NT, LISTS>::kCTAs) quant_rows_kernel(const QuantArgs a, const int row_tiles) {
    using Sh = QuantShape<D, NT, LISTS>;
    constexpr int kRows = 8 * NT;
    constexpr int C = D / 16;       // 16-byte chunks of a key
    constexpr int KS = D / 16;      // k-steps of S
    constexpr int MT = D / 16;      // M tiles of O
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, c = lane & 3;
    if (a.cluster) cluster_arrive();
    grid_wait();
    grid_trigger();
    // (parts, KV heads x row tiles, sequences)
    const int split = blockIdx.x, b = blockIdx.z;
    const int h = row_tiles == 1 ? (int)blockIdx.y : (int)blockIdx.y / row_tiles;
    const int r0 = ((int)blockIdx.y - h * row_tiles) * kRows;
    const int nrows = a.Tq * a.G;
    const int live = nrows - r0 < kRows ? nrows - r0 : kRows;
    // Q's rows are asked for before what the lengths say is known: row r0 + g (and + 8); k-step kk's four values of a
    // lane are D's 16 (c + 4 (kk / 4)) + 4 (kk % 4) + 0..3
    constexpr bool kShared = NT == 4;
    constexpr int NQ = kShared ? 1 : NT;
    uint32_t qf[NQ][KS][2];  // as they are, then as halves
#pragma unroll
    for (int u = 0; u < NQ; ++u) {
        const int r = r0 + g + 8 * (kShared ? warp : u), tok = token_of(a, r);
        const T* src = static_cast<const T*>(a.q) + b * a.q_b + tok * a.q_t + (h * (int64_t)a.G + r - tok * a.G) * a.q_h;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
            const uint2 raw = r < nrows ? *reinterpret_cast<const uint2*>(src + 16 * (c + 4 * (kk >> 2)) + 4 * (kk & 3))
                                        : make_uint2(0, 0);
            qf[u][kk][0] = raw.x, qf[u][kk][1] = raw.y;
        }
    }
    // keys: positions of the sequence, or entries of the list
    int trow = b, length, keys;
    if (LISTS) {
        trow = a.list_rows ? a.list_rows[b] : b;
        const bool ok = trow >= 0 && trow < a.table_rows;
        trow = ok ? trow : 0;
        length = ok ? max(a.lengths[trow], 0) : 0;
        keys = a.counts[b];
        keys = !ok || keys < 0 ? 0 : (keys > a.W ? a.W : keys);
    } else {
        length = max(a.lengths[b], 0);
        keys = length - a.Tq + token_of(a, r0 + live - 1) + 1;  // that the tile's last row sees
        const int64_t room = (int64_t)a.M << a.shift;
        keys = keys < 0 ? 0 : (keys > room ? (int)room : keys);
    }
    int k0, k1;
    {
        // a list is split by its width: its entries are asked for beside its count
        const int64_t units = ((LISTS ? a.W : keys) + kWarps * kKeys - 1) / (kWarps * kKeys);
        const int64_t u0 = units * split / a.parts * (kWarps * kKeys), u1 = units * (split + 1) / a.parts * (kWarps * kKeys);
        const int all = LISTS ? a.W : keys;
        k0 = (int)(u0 < all ? u0 : all), k1 = (int)(u1 < all ? u1 : all);
    }
    const int32_t* table = a.table + trow * a.table_ld;
    const int32_t* list = LISTS ? a.lists + (int64_t)b * a.W : nullptr;
    const uint32_t ring = smem_u32(smem) + warp * Sh::kWarpBytes;
    const int tiles = k1 - k0 > warp * kKeys ? (k1 - k0 - warp * kKeys + kWarps * kKeys - 1) / (kWarps * kKeys) : 0;

    // Tile i of this warp: keys k0 + (warp + 4 i) 32 ..; a lane looks its key up, two tiles ahead the position, one
    // the page; then the warp copies the rows.
    auto position = [&](int i) {
        const int key = k0 + (warp + kWarps * i) * kKeys + lane;
        const bool in = i < tiles && key < k1;
        const int pos = !in ? -1 : (LISTS ? list[key] : key);
        return LISTS && key >= keys ? -1 : pos;
    };
    auto page_of = [&](int pos) {
        return pos >= 0 && pos < length && (pos >> a.shift) < a.M ? table[pos >> a.shift] : -1;
    };
    // row of the pool (below 2^31: the entry point checks) of a position; a key that is not there is not read
    auto row_of = [&](int pos, int page) {
        return page >= 0 && page < a.pages
                   ? (int)((((int64_t)page * a.Hkv + h) << a.shift) + (pos & ((1 << a.shift) - 1)))
                   : -1;
    };
    int pos1 = position(0), pos2 = position(1), page1 = page_of(pos1);
    uint32_t there = 0;  // bit j: this lane's key of the j-th tile before the last copied is there
    const uint8_t* const kl = a.k8 + (lane / C) * D + (lane % C) * 16;
    const uint8_t* const vl = a.v8 + (lane / C) * D + (lane % C) * 16;
    uint32_t slot = 0;  // of the next copy
    auto copy = [&](int i) {
        const int row = row_of(pos1, page1);
        pos1 = pos2, page1 = page_of(pos2), pos2 = position(i + 2);
        there <<= 1;
        if (i < tiles) {
            const bool in = row >= 0;
            there |= in ? 1u : 0u;
            const int64_t head = in ? row >> a.shift : 0;
            const uint32_t stage = ring + slot * Sh::kStage;
            const uint32_t scales = stage + 2 * Sh::kTile + lane * 4;
            cp_async4(scales, a.ks + head, in ? 4u : 0u);
            cp_async4(scales + kKeys * 4, a.vs + head, in ? 4u : 0u);
            if (LISTS) {
#pragma unroll
                for (int rr = 0; rr < kKeys; rr += 32 / C) {
                    const int r = rr + lane / C, ch = lane % C;
                    const int from = __shfl_sync(0xFFFFFFFFu, row, r);
                    const int64_t at = (int64_t)((from < 0 ? 0 : from) - lane / C) * D;
                    cp_async16(stage + k_at<D>(r, ch), from < 0 ? a.k8 : kl + at, from < 0 ? 0u : 16u);
                    cp_async16(stage + Sh::kTile + v_at<D>(r, ch), from < 0 ? a.v8 : vl + at, from < 0 ? 0u : 16u);
                }
            } else {
                // 16 keys lie on one page: their rows follow one another, and the last ones may be past k1
                const uint32_t live = __ballot_sync(0xFFFFFFFFu, in);
                const int from = __shfl_sync(0xFFFFFFFFu, row, 0), from2 = __shfl_sync(0xFFFFFFFFu, row, 16);
                const int64_t at = (int64_t)(from < 0 ? 0 : from) * D, at2 = (int64_t)(from2 < 0 ? 0 : from2) * D;
                const uint8_t *kp = kl + at, *vp = vl + at, *kp2 = kl + at2 - 16 * D, *vp2 = vl + at2 - 16 * D;
                const uint32_t kd = stage + k_at<D>(lane / C, lane % C);
                if (live == 0xFFFFFFFFu) {
#pragma unroll
                    for (int rr = 0; rr < kKeys; rr += 32 / C) {
                        cp_async16_all(kd + rr * D, (rr < 16 ? kp : kp2) + rr * D);
                        cp_async16_all(stage + Sh::kTile + v_at<D>(rr + lane / C, lane % C), (rr < 16 ? vp : vp2) + rr * D);
                    }
                } else {
#pragma unroll
                    for (int rr = 0; rr < kKeys; rr += 32 / C) {
                        const bool one = live >> (rr + lane / C) & 1u;
                        cp_async16(kd + rr * D, one ? (rr < 16 ? kp : kp2) + rr * D : a.k8, one ? 16u : 0u);
                        cp_async16(stage + Sh::kTile + v_at<D>(rr + lane / C, lane % C),
                                   one ? (rr < 16 ? vp : vp2) + rr * D : a.v8, one ? 16u : 0u);
                    }
                }
            }
        }
        if (++slot == Sh::kRing) slot = 0;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // Q's fragments, as halves
    uint64_t factor[NT];  // of rows r0 + 2c and 2c + 1 (and + 8), as the maxima and sums below
    int limit[NT][2];
    const uint32_t qs = smem_u32(smem + Sh::kQ), fs = qs + kRows * D * 2;
    auto prepare = [&]() {
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
            float f = a.scale_log2;
            uint32_t top = 0;  // largest magnitude's bits
#pragma unroll
            for (int kk = 0; kk < KS; ++kk)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    top = max(top, max(qf[u][kk][e] & 0x7FFFu, (qf[u][kk][e] >> 16) & 0x7FFFu));
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                const float by = half_factor(top, &f);
#pragma unroll
                for (int kk = 0; kk < KS; ++kk)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        qf[u][kk][e] = pack_half(__uint_as_float(qf[u][kk][e] << 16) * by,
                                                 __uint_as_float(qf[u][kk][e] & 0xFFFF0000u) * by);
            }
            if (infinite_row<T>(top)) {
                f = kInfiniteRow;
#pragma unroll
                for (int kk = 0; kk < KS; ++kk) qf[u][kk][0] = qf[u][kk][1] = 0;
            }
            if constexpr (kShared) {
#pragma unroll
                for (int kk = 0; kk < KS; ++kk)
                    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(qs + ((kk * NT + warp) * 32 + lane) * 8),
                                 "r"(qf[u][kk][0]), "r"(qf[u][kk][1])
                                 : "memory");
                if (c == 0) sts_f32(fs + (warp * 8 + g) * 4, f);
            } else {
                factor[u] = pair(__shfl_sync(0xFFFFFFFFu, f, 8 * c), __shfl_sync(0xFFFFFFFFu, f, 8 * c + 4));
            }
        }
        if constexpr (kShared) __syncthreads();
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            if constexpr (kShared) factor[u] = lds64(fs + (8 * u + 2 * c) * 4);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = r0 + 8 * u + 2 * c + e;
                limit[u][e] = row >= nrows ? 0 : length - a.Tq + token_of(a, row) + 1;
            }
        }
    };
    if (kShared) prepare();  // by all warps; else behind the first copies
    const int first_limit = length - a.Tq + token_of(a, r0) + 1;  // keys that the tile's first row sees
    float o[NT][MT][4];  // O^T: columns (D / 8) g + 2 j (0, 1) and + 1 (2, 3) of rows 2c (0, 2) and 2c + 1 (1, 3)
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[u][j][e] = 0.0f;
    float m[NT][2];
    uint64_t l[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) m[u][0] = m[u][1] = -INFINITY, l[u] = 0ull;

    uint32_t read = 0;  // slot of tile i
    // one copy of the code that copies: a launch starts with it cold
#pragma unroll 1
    for (int i = 1 - Sh::kRing; i < tiles; ++i) {
        copy(i + Sh::kRing - 1);
        if (i < 0) continue;
        if (!kShared && i == 0) prepare();
        asm volatile("cp.async.wait_group %0;" ::"n"(Sh::kRing - 1) : "memory");
        const uint32_t ks = ring + read * Sh::kStage, vs = ks + Sh::kTile, scales = vs + Sh::kTile;
        if (++read == Sh::kRing) read = 0;
        const int key0 = k0 + (warp + kWarps * i) * kKeys;
        // this lane's key: vs becomes its logarithm, -inf where there is no key, and its inverse
        {
            const bool in = there >> (Sh::kRing - 1) & 1u;
            const float v = fmaxf(__uint_as_float(lds32(scales + kKeys * 4 + lane * 4)), 8.6736174e-19f);  // 2^-60
            sts_f32(scales + kKeys * 4 + lane * 4, in ? lg2_approx(v) : -INFINITY);
            sts_f32(scales + kKeys * 8 + lane * 4, in ? rcp_approx(v) : 0.0f);
        }
        __syncwarp();
        // logits x[u][k]: key 8 k + g, rows 2c and 2c + 1, with the value scale in the exponent; -inf where there is no
        // key, or none for the row
        uint64_t x[NT][4];
        if constexpr (!kShared) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                float s[NT][4];
#pragma unroll
                for (int u = 0; u < NT; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[u][e] = 0.0f;
#pragma unroll
                for (int hh = 0; hh < KS / 4; ++hh) {
                    uint32_t w0[4], w1[4];
                    lds_words<4>(w0, ks + k_at<D>(t * 16 + g, c + 4 * hh));
                    lds_words<4>(w1, ks + k_at<D>(t * 16 + 8 + g, c + 4 * hh));
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        const uint32_t kf[4] = {halves_of<CODE>(w0[kk], 0), halves_of<CODE>(w1[kk], 0),
                                                halves_of<CODE>(w0[kk], 1), halves_of<CODE>(w1[kk], 1)};
#pragma unroll
                        for (int u = 0; u < NT; ++u) mma_f16(s[u], kf, qf[u][4 * hh + kk][0], qf[u][4 * hh + kk][1]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int u = 0; u < NT; ++u) x[u][2 * t + e] = pair(s[u][2 * e], s[u][2 * e + 1]);
            }
        } else {
            float s[2][NT][4];
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[0][u][e] = s[1][u][e] = 0.0f;
#pragma unroll
            for (int hh = 0; hh < KS / 4; ++hh) {
                uint32_t w[4][4];
#pragma unroll
                for (int y = 0; y < 4; ++y) lds_words<4>(w[y], ks + k_at<D>(y * 8 + g, c + 4 * hh));
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    uint32_t kf[2][4];
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) kf[t][e] = halves_of<CODE>(w[2 * t + (e & 1)][kk], e >> 1);
#pragma unroll
                    for (int u = 0; u < NT; ++u) {
                        uint32_t q[2];
                        lds_words<2>(q, qs + (((4 * hh + kk) * NT + u) * 32 + lane) * 8);
                        mma_f16(s[0][u], kf[0], q[0], q[1]);
                        mma_f16(s[1][u], kf[1], q[0], q[1]);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k) x[u][k] = pair(s[k >> 1][u][2 * (k & 1)], s[k >> 1][u][2 * (k & 1) + 1]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t at = scales + (k * 8 + g) * 4;
            const float key_scale = __uint_as_float(lds32(at)), lv = __uint_as_float(lds32(at + kKeys * 4));
#pragma unroll
            for (int u = 0; u < NT; ++u)
                x[u][k] = fma2(mul2(x[u][k], pair(key_scale, key_scale)), factor[u], pair(lv, lv));
        }
        if (!LISTS && key0 + kKeys > first_limit) {  // rows before the tile's last see less
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float x0, x1;
                    unpair(x[u][k], x0, x1);
                    const int key = key0 + 8 * k + g;
                    x[u][k] = pair(key < limit[u][0] ? x0 : -INFINITY, key < limit[u][1] ? x1 : -INFINITY);
                }
        }
        float mx[NT][2];
        bool grow = false;
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            float y[4][2];
#pragma unroll
            for (int k = 0; k < 4; ++k) unpair(x[u][k], y[k][0], y[k][1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float v = fmaxf(max3(y[0][e], y[1][e], y[2][e]), y[3][e]);
#pragma unroll
                for (int off = 4; off <= 16; off <<= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, off));
                mx[u][e] = v;
                grow = grow || v > m[u][e] + kGrow;  // m = -inf: any key
            }
        }
        if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                float alpha[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float mn = fmaxf(m[u][e], mx[u][e]);
                    alpha[e] = mn == -INFINITY ? 0.0f : ex2_approx(m[u][e] - mn);
                    m[u][e] = mn;
                }
                const uint64_t al = pair(alpha[0], alpha[1]);
                l[u] = mul2(l[u], al);
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    unpair(mul2(pair(o[u][j][0], o[u][j][1]), al), o[u][j][0], o[u][j][1]);
                    unpair(mul2(pair(o[u][j][2], o[u][j][3]), al), o[u][j][2], o[u][j][3]);
                }
            }
        }
        uint32_t p[NT][4];  // P^T's fragments: row g, keys 8 k + 2c and + 1
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            const uint64_t neg = pair(m[u][0] == -INFINITY ? 0.0f : -m[u][0], m[u][1] == -INFINITY ? 0.0f : -m[u][1]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float x0, x1;
                unpair(add2(add2(x[u][k], neg), pair(kLift, kLift)), x0, x1);
                const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
                const float inv = __uint_as_float(lds32(scales + kKeys * 8 + (8 * k + g) * 4));
                l[u] = fma2(pair(p0, p1), pair(inv, inv), l[u]);
                p[u][k] = transposed(pack_half(p0, p1));
            }
        }
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            // keys 16 kk + 2c, + 1, + 8, + 9 of the tile
            constexpr int NW = D / 32;  // words of a key a lane takes: D's (D / 8) g ..
            uint32_t w[4][NW];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 16 * kk + 2 * c + (i & 1) + 8 * (i >> 1);
                if constexpr (D == 128)
                    lds_words<NW>(w[i], vs + v_at<D>(r, g));
                else
                    lds_words<NW>(w[i], vs + v_at<D>(r, g >> 1) + (g & 1) * 8);
            }
#pragma unroll
            for (int j = 0; j < 2 * NW; ++j) {
                const uint32_t sel = j & 1 ? 0x7362 : 0x5140;
                const uint32_t lo = __byte_perm(w[0][j >> 1], w[1][j >> 1], sel), hi = __byte_perm(w[2][j >> 1], w[3][j >> 1], sel);
                const uint32_t vf[4] = {halves_of<CODE>(lo, 0), halves_of<CODE>(lo, 1), halves_of<CODE>(hi, 0),
                                        halves_of<CODE>(hi, 1)};
#pragma unroll
                for (int u = 0; u < NT; ++u) mma_f16(o[u][j], vf, p[u][2 * kk], p[u][2 * kk + 1]);
            }
        }
        __syncwarp();  // the tile's slot is refilled next
    }
    cp_async_wait_all();
    float sum[NT][2];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
        unpair(l[u], sum[u][0], sum[u][1]);
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int off = 4; off <= 16; off <<= 1) sum[u][e] += __shfl_xor_sync(0xFFFFFFFFu, sum[u][e], off);
        float f[2];
        unpair(factor[u], f[0], f[1]);
#pragma unroll
        for (int e = 0; e < 2; ++e) sum[u][e] = sum_of_row(sum[u][e], f[e]);
    }
    // join the warps: each leaves its sums in its own ring, (m, l) after the rings
    __syncwarp();
    float* so = reinterpret_cast<float*>(smem + warp * Sh::kWarpBytes);
    float2* sml = reinterpret_cast<float2*>(smem + kWarps * Sh::kWarpBytes);
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = 8 * u + 2 * c + e;
            float* line = so + r * D + (D / 8) * g;
#pragma unroll
            for (int j = 0; j < MT; j += 2)
                *reinterpret_cast<float4*>(line + 2 * j) =
                    make_float4(o[u][j][e], o[u][j][2 + e], o[u][j + 1][e], o[u][j + 1][2 + e]);
            if (g == 0) sml[warp * kRows + r] = make_float2(m[u][e], sum[u][e]);
        }
    __syncthreads();
    auto row_id = [&](int r) {
        const int tok = token_of(a, r0 + r);
        return ((int64_t)b * a.Tq + tok) * a.Hq + (int64_t)h * a.G + (r0 + r - tok * a.G);
    };
    if (a.cluster) cluster_wait();  // every CTA of the cluster runs: its memory may be written
    for (int i = threadIdx.x; i < live * (D / 4); i += kWarps * 32) {
        const int r = i / (D / 4), col = i % (D / 4) * 4;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sml[w * kRows + r].x);
        float total = 0.0f;
        float4 x = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float2 ml = sml[w * kRows + r];
            const float f = ml.y == 0.0f ? 0.0f : ex2_approx(ml.x - top);  // NaN passes on
            const float4 y = *reinterpret_cast<const float4*>(smem + w * Sh::kWarpBytes + (r * D + col) * 4);
            total = fmaf(f, ml.y, total);
            x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y), x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w);
        }
        const float norm = total == 0.0f ? 0.0f : 1.0f / total;
        x.x *= norm, x.y *= norm, x.z *= norm, x.w *= norm;
        const float lse = total == 0.0f ? -INFINITY : top + (log2f(total) - kLift);
        if (a.cluster) {  // to the CTA that joins these columns: every parts-th item, in the sender's place
            const int to = i & (a.parts - 1), at = split * (live * (D / 4) / a.parts) + i / a.parts;
            send_f4(peer(smem_u32(smem + Sh::kIn) + at * 16, to), x);
            send_f1(peer(smem_u32(smem + Sh::kIn) + Sh::kItems * 16 + at * 4, to), lse);
            continue;
        }
        const int64_t rid = row_id(r);
        if (a.parts == 1) {
            store4<T>(static_cast<T*>(a.out) + rid * D + col, x);
            if (col == 0 && a.lse) a.lse[rid] = lse * 0.69314718055994531f;
        } else {
            const int64_t at = (int64_t)split * a.part_rows + rid;
            *reinterpret_cast<float4*>(a.part_o + at * D + col) = x;
            if (col == 0) a.part_lse[at] = lse;
        }
    }
    if (!a.cluster) return;
    __syncwarp();
    // A cluster holds all parts of its rows: every CTA has the others' sums of its own columns once all have arrived.
    cluster_arrive();
    cluster_wait();
    const int per = live * (D / 4) / a.parts;
    for (int j = threadIdx.x; j < per; j += kWarps * 32) {
        const int i = j * a.parts + split, r = i / (D / 4), col = i % (D / 4) * 4;
        float top = -INFINITY, total = 0.0f, lse[kMostCluster];
        float4 x = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int p = 0; p < kMostCluster; ++p) {
            lse[p] = p < a.parts ? *reinterpret_cast<const float*>(smem + Sh::kIn + Sh::kItems * 16 + (p * per + j) * 4) : -INFINITY;
            top = fmaxf(top, lse[p]);
        }
#pragma unroll
        for (int p = 0; p < kMostCluster; ++p) {
            if (p >= a.parts) break;
            const float4 y = *reinterpret_cast<const float4*>(smem + Sh::kIn + (p * per + j) * 16);
            const float f = lse[p] == -INFINITY ? 0.0f : ex2_approx(lse[p] - top);  // NaN passes on
            total += f;
            x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y), x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w);
        }
        const float norm = total == 0.0f ? 0.0f : 1.0f / total;
        const int64_t rid = row_id(r);
        store4<T>(static_cast<T*>(a.out) + rid * D + col, make_float4(x.x * norm, x.y * norm, x.z * norm, x.w * norm));
        if (col == 0 && a.lse) a.lse[rid] = total == 0.0f ? -INFINITY : (top + log2f(total)) * 0.69314718055994531f;
    }
}

// The parts of a row joined, SPREAD warps a row (one where the parts are few, so that a CTA takes eight rows). Every
// part's values are asked for before the weights are known, so a row is one round of memory.
template <typename T, int D, int SPREAD>
__global__ void __launch_bounds__(256) quant_join_kernel(const QuantArgs a, const int parts) {
    constexpr int V = D / 32, N = SPREAD == 1 ? kFewParts : kMaxQuantParts / SPREAD;
    constexpr int L = SPREAD == 1 ? 1 : kMaxQuantParts / 32;  // loads of the parts' sums, 32 each
    __shared__ float so[8][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % SPREAD;
    grid_wait();
    grid_trigger();
    const int64_t prow = (int64_t)blockIdx.x * (8 / SPREAD) + warp / SPREAD;
    int64_t rid = prow;
    bool live = prow < a.part_rows;
    if (a.tokens > 0 && live) {  // the rows of the split tiles
        const int per = quant_tile_rows(a.streams), rl = (int)(prow % per), hf = rl >> 7;
        int b, h, tile;
        quant_tile_at(a, a.whole + (int)(prow / per), &b, &h, &tile);
        const int tl = (rl & 127) / a.G, tok = tile * (per / 128) * a.tokens + hf * a.tokens + tl;
        live = tl < a.tokens && tok < a.Tq;
        rid = ((int64_t)b * a.Tq + tok) * a.Hq + (int64_t)h * a.G + (rl & 127) - tl * a.G;
    }
    float lse[L], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < L; ++i) {
        const int part = i * 32 + lane;
        lse[i] = live && part < parts ? a.part_lse[part * a.part_rows + prow] : -INFINITY;
    }
    float y[N][V];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int part = sub + SPREAD * i;
        const float* src = a.part_o + (part * a.part_rows + prow) * D + lane * V;
#pragma unroll
        for (int e = 0; e < V; ++e) y[i][e] = 0.0f;
        if (live && part < parts) {
            if constexpr (V == 4) {
                const float4 z = *reinterpret_cast<const float4*>(src);
                y[i][0] = z.x, y[i][1] = z.y, y[i][2] = z.z, y[i][3] = z.w;
            } else {
                const float2 z = *reinterpret_cast<const float2*>(src);
                y[i][0] = z.x, y[i][1] = z.y;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < L; ++i) top = fmaxf(top, lse[i]);
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, off));
    float total = 0.0f, f[L], o[V];
#pragma unroll
    for (int i = 0; i < L; ++i) {  // NaN passes on
        f[i] = lse[i] == -INFINITY ? 0.0f : exp2f(lse[i] - (top == -INFINITY ? 0.0f : top));
        total += f[i];
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, off);
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float fi = __shfl_sync(0xFFFFFFFFu, f[SPREAD * i / 32], (sub + SPREAD * i) & 31);
        // what a part without a key holds is never used
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = fi == 0.0f ? o[e] : fmaf(fi, y[i][e], o[e]);
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    if constexpr (SPREAD == 1) {
        if (live) {
            T* dst = static_cast<T*>(a.out) + rid * D + lane * V;
            if constexpr (V == 4)
                store4<T>(dst, make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv));
            else
                *reinterpret_cast<uint32_t*>(dst) = pack16(o[0] * inv, o[1] * inv, (T*)nullptr);
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) so[warp][lane * V + e] = o[e];
        __syncthreads();
        const int col = threadIdx.x;
        if (col < D && live) {
            float x = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) x += so[w][col];
            static_cast<T*>(a.out)[rid * D + col] = from_f32<T>(x * inv);
        }
    }
    if (lane == 0 && sub == 0 && live && a.lse)
        a.lse[rid] = total == 0.0f ? -INFINITY : (top + log2f(total)) * 0.69314718055994531f;
}

template <typename T, int CODE, int D, bool LISTS, int NT>
int launch(const QuantArgs& a, int row_tiles, dim3 grid, cudaStream_t stream) {
    // A grid of one round on two places an SM takes so much shared memory that no SM has a third: its CTAs start while
    // those of the launch before leave, and would gather where places are free first (4 x 16k keys 28.8 us, so 24.4).
    constexpr int least = QuantShape<D, NT, LISTS>::kSmem, two = 100 << 10;
    const int smem = (int64_t)grid.x * grid.y * grid.z <= 2 * 148 && least < two ? two : least;
    if (!allow_kernel<quant_rows_kernel<T, CODE, D, LISTS, NT>>(least < two ? two : least, true)) return LSA_ERR_CUDA;
    return launch_clusters(quant_rows_kernel<T, CODE, D, LISTS, NT>, grid, kWarps * 32, smem, stream,
                           a.cluster ? a.parts : 1, a, row_tiles);
}
template <typename T, int CODE, int D>
int launch(const QuantArgs& a, int row_tiles, dim3 grid, cudaStream_t stream) {
    const int rows = a.Tq * a.G;
    if (a.lists)
        return rows <= 8 ? launch<T, CODE, D, true, 1>(a, row_tiles, grid, stream)
                         : launch<T, CODE, D, true, 2>(a, row_tiles, grid, stream);
    if (rows > 16) return launch<T, CODE, D, false, 4>(a, row_tiles, grid, stream);
    return rows <= 8 ? launch<T, CODE, D, false, 1>(a, row_tiles, grid, stream)
                     : launch<T, CODE, D, false, 2>(a, row_tiles, grid, stream);
}
template <typename T> int launch(const QuantArgs& a, int code, int D, int row_tiles, dim3 grid, cudaStream_t stream) {
    if (code == kE4M3)
        return D == 128 ? launch<T, kE4M3, 128>(a, row_tiles, grid, stream) : launch<T, kE4M3, 64>(a, row_tiles, grid, stream);
    return D == 128 ? launch<T, kInt8, 128>(a, row_tiles, grid, stream) : launch<T, kInt8, 64>(a, row_tiles, grid, stream);
}

}  // namespace

int launch_quant_rows(const QuantArgs& a, int dtype, int code, int D, cudaStream_t stream) {
    const int64_t tiles = few_row_tiles((int64_t)a.Tq * a.G, a.lists != nullptr);
    if (a.B > 65535 || a.Hkv * tiles > 65535) return LSA_ERR_SIZE;
    const int row_tiles = (int)tiles;
    const dim3 grid((unsigned)a.parts, (unsigned)(a.Hkv * row_tiles), (unsigned)a.B);
    return dtype == kBF16 ? launch<__nv_bfloat16>(a, code, D, row_tiles, grid, stream)
                          : launch<__half>(a, code, D, row_tiles, grid, stream);
}

template <typename T, int D> static int join(const QuantArgs& a, cudaStream_t stream) {
    const int parts = a.tokens > 0 && a.streams ? 2 * a.parts : a.parts;
    const int64_t blocks = parts <= kFewParts ? (a.part_rows + 7) / 8 : a.part_rows;
    if (blocks > INT32_MAX || parts > kMaxQuantParts) return LSA_ERR_SIZE;
    const dim3 grid((unsigned)blocks);
    return parts <= kFewParts ? launch_after(quant_join_kernel<T, D, 1>, grid, 256, 0, stream, a, parts)
                              : launch_after(quant_join_kernel<T, D, 8>, grid, 256, 0, stream, a, parts);
}

int launch_quant_join(const QuantArgs& a, int dtype, int D, cudaStream_t stream) {
    if (dtype == kBF16) return D == 128 ? join<__nv_bfloat16, 128>(a, stream) : join<__nv_bfloat16, 64>(a, stream);
    return D == 128 ? join<__half, 128>(a, stream) : join<__half, 64>(a, stream);
}

}  // namespace lsa
