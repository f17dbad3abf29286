// evict.cu - eviction from a KV cache by accumulated attention weight (sm_100a).
//
// For sequence b with n keys and KV head h: n <= budget keeps every key; else the sinks
// [0, sink), the window [n - window, n) and, of the keys between, the budget - sink - window
// with the highest score stay. Scores order as the selection's packed keys do (ordered_bits:
// -NaN < -inf < ... < -0 < +0 < ... < +inf < +NaN), ties go to the lower index. The kept keys
// keep their order: out slot m holds kept key ids[m], ascending; slots past the kept count are
// zeros (ids -1).
#include "launch.cuh"

namespace lsa {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;     // 11 bits a pass: 3 passes over 32-bit keys
constexpr int kCached = 16384;  // keys held in a CTA's shared memory (more are read again)

struct EvictArgs {
    const void *k, *v;
    int64_t k_b, k_t, k_h, v_b, v_t, v_h;  // strides in bytes
    const float* scores;                   // [B, Hkv, T]
    const int32_t* lengths;                // [B]
    int B, T, Hkv, row_bytes, row_lanes;
    int budget, window, sink, capacity;
    bool copy;                             // the selecting kernel copies the rows too
    void *k_out, *v_out;                   // [B, capacity, Hkv, D] contiguous
    float* scores_out;                     // [B, Hkv, capacity]
    int32_t* lengths_out;                  // [B]
    int32_t* ids;                          // [B, Hkv, capacity]
};

__device__ __forceinline__ uint32_t score_key(float f) { return (uint32_t)ordered_bits(f) ^ 0x80000000u; }

__device__ __forceinline__ float key_score(uint32_t u) {  // the score itself again, bit for bit
    const int32_t o = (int32_t)(u ^ 0x80000000u);
    return __int_as_float(o >= 0 ? o : o ^ 0x7FFFFFFF);
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the address, in the cluster's shared memory, of `p` in CTA `rank`
__device__ __forceinline__ uint32_t at_rank(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ int4 ld_cluster4(uint32_t addr) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

__device__ __forceinline__ void add_cluster(uint32_t addr, int v) {
    if (v) asm volatile("red.relaxed.cluster.shared::cluster.add.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// The rows of K and V of slots [m0, m1) by their ids: a row of 16-byte chunks to the next power of
// two of lanes (at most a warp), four rows a thread in flight; zeros for a slot without an id.
__device__ __forceinline__ void copy_rows(const EvictArgs& a, int b, int h, int m0, int m1) {
    const int32_t* ids = a.ids + ((int64_t)b * a.Hkv + h) * a.capacity;
    const int tid = threadIdx.x;
    const int chunks = a.row_bytes >> 4, lanes = a.row_lanes;
    const int sub = tid / lanes, step = kThreads / lanes;
    const uint8_t* kb = static_cast<const uint8_t*>(a.k) + b * a.k_b + h * a.k_h;
    const uint8_t* vb = static_cast<const uint8_t*>(a.v) + b * a.v_b + h * a.v_h;
    const int64_t out_t = (int64_t)a.Hkv * a.row_bytes;
    uint8_t* ko = static_cast<uint8_t*>(a.k_out) + ((int64_t)b * a.capacity * a.Hkv + h) * a.row_bytes;
    uint8_t* vo = static_cast<uint8_t*>(a.v_out) + ((int64_t)b * a.capacity * a.Hkv + h) * a.row_bytes;
    for (int c = tid % lanes; c < chunks; c += lanes) {
        for (int m = m0 + sub; m < m1; m += 4 * step) {
            uint4 x[4], y[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int mu = m + u * step;
                const int id = mu < m1 ? ids[mu] : -1;
                x[u] = y[u] = make_uint4(0, 0, 0, 0);
                if (id >= 0) {
                    x[u] = __ldg(reinterpret_cast<const uint4*>(kb + id * a.k_t) + c);
                    y[u] = __ldg(reinterpret_cast<const uint4*>(vb + id * a.v_t) + c);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int mu = m + u * step;
                if (mu < m1) {
                    reinterpret_cast<uint4*>(ko + mu * out_t)[c] = x[u];
                    reinterpret_cast<uint4*>(vo + mu * out_t)[c] = y[u];
                }
            }
        }
    }
}

// Every row (sequence, KV head) is served by `ranks` CTAs.
//  1. The last score that stays: a radix search over the competing keys, 11 bits a pass from the
//     top; it ends early when all keys of a bin stay.
//  2. Output slots from kept counts, by warp ballots, in index order: ids and scores.
//  3. The kept rows of K and V are copied, every CTA an equal share of the output slots whoever
//     selected them (heavy keys crowd together: the sinks, the window).
// kSliced false: every CTA of a row selects over all its keys by itself, without a word to the
// others - the selection is latency, not work, while its keys fit one CTA's shared memory. true: the
// CTAs are a cluster, hold a slice of the keys each, and join their histograms (DSMEM adds into the
// bins' owner, one cluster barrier a pass) and their kept counts.
// Selection is a chain of short steps, the copy is bandwidth: with several CTAs an SM one row's
// copy covers another's chain. Measured (D 128, bf16, called in a loop): 64 ragged caches of up to 8191 keys, 8
// heads, to 2048: 187 us = 5.9 TB/s; 4 of 131072 to 8192: 72 us, of which the selection takes about 23 (the
// rows are in lock-step: 256 CTAs, 32 keys a thread) and 268 MB of copying the rest; one of 2112 to 2048: 12 us
// (the host's), the kernel alone 9.6, 7 of them selection (load 1.9, a pass 1.1, counts and ids 1.7).
template <bool kSliced>
__global__ void __launch_bounds__(kThreads, 2) evict_kernel(const EvictArgs a, int ranks_arg) {
    __shared__ __align__(16) int hist[kBins];
    __shared__ __align__(16) int joined[kSliced ? 3 * kBins / 2 : 4];  // this rank's bins, one set a pass
    __shared__ int scan[kWarps], wkeep[kWarps], wtie[kWarps];
    __shared__ __align__(16) int4 found;   // digit, keys still needed, keys of the digit
    __shared__ __align__(16) int4 counts;  // keys of the slice that stay for sure, and on the level
    extern __shared__ uint32_t keys[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int ranks = ranks_arg, rank = blockIdx.x % ranks;  // the cluster rank, when sliced
    const int row = blockIdx.x / ranks, h = row % a.Hkv, b = row / a.Hkv;
    int n = a.lengths[b];
    n = n < 0 ? 0 : (n > a.T ? a.T : n);
    const int kept = n < a.budget ? n : a.budget;
    const float* sc = a.scores + ((int64_t)b * a.Hkv + h) * a.T;
    int32_t* ids = a.ids + ((int64_t)b * a.Hkv + h) * a.capacity;
    float* so = a.scores_out + ((int64_t)b * a.Hkv + h) * a.capacity;
    if (h == 0 && rank == 0 && tid == 0) a.lengths_out[b] = kept;
    // the output's slots, an equal share a CTA
    const int m0 = (int)((int64_t)a.capacity * rank / ranks), m1 = (int)((int64_t)a.capacity * (rank + 1) / ranks);

    if (n > a.budget) {
        const int s0 = kSliced ? (int)((int64_t)n * rank / ranks) : 0;
        const int s1 = kSliced ? (int)((int64_t)n * (rank + 1) / ranks) : n;
        const int lo = a.sink, hi = n - a.window;  // the keys that compete
        auto key_at = [&](int j) {
            if (!kSliced) return keys[j];
            return j - s0 < kCached ? keys[j - s0] : score_key(sc[j]);
        };
        int need = a.budget - a.sink - a.window;
        // a key stays when its top bits are above `cut`; on the level, the first `level` by index
        uint32_t cut = 0;
        int shift = 0, level = 0;
        // warp w owns the keys [w0, w1), a lane every 32nd; loads go in groups at clamped indices, so
        // that a group's are all in flight
        const int seg = ((s1 - s0 + 31) / 32 + kWarps - 1) / kWarps * 32;
        const int w0 = s0 + warp * seg < s1 ? s0 + warp * seg : s1, w1 = w0 + seg < s1 ? w0 + seg : s1;
        for (int j0 = w0; j0 < w1 && j0 - s0 < kCached; j0 += 32 * 16) {
            float x[16];
#pragma unroll
            for (int u = 0; u < 16; ++u) {
                const int j = j0 + 32 * u + lane;
                x[u] = __ldg(sc + (j < w1 ? j : w1 - 1));
            }
#pragma unroll
            for (int u = 0; u < 16; ++u) {
                const int j = j0 + 32 * u + lane;
                if (j < w1 && j - s0 < kCached) keys[j - s0] = score_key(x[u]);
            }
        }
        // f(j, key) for the warp's keys, 32 consecutive ones a step (j at or past w1: no key)
        auto each = [&](auto f) {
            int j = w0 + lane;
            for (; j - lane + 128 <= (w1 < s0 + kCached ? w1 : s0 + kCached); j += 128) {
                uint32_t u[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) u[q] = keys[j - s0 + 32 * q];
#pragma unroll
                for (int q = 0; q < 4; ++q) f(j + 32 * q, u[q]);
            }
#pragma unroll 1
            for (; j - lane < w1; j += 32) f(j, j < w1 ? key_at(j) : 0u);
        };
        if (kSliced) {
            for (int i = tid; i < 3 * kBins / 2; i += kThreads) joined[i] = 0;
            cluster_sync();
        }
        if (need == 0) {
            cut = 0xFFFFFFFFu;
            __syncthreads();
        } else {
            shift = 32;
#pragma unroll
            for (int pass = 0; pass < 3; ++pass) {
                const int width = pass == 2 ? 10 : 11, up = shift;
                shift -= width;
                *reinterpret_cast<int4*>(hist + 4 * tid) = make_int4(0, 0, 0, 0);
                __syncthreads();
                const int end = s1 < hi ? s1 : hi;
                auto count = [&](uint32_t u) {
                    if (pass == 0 || (u >> up) == cut) atomicAdd(&hist[(u >> shift) & ((1u << width) - 1)], 1);
                };
                int j = (s0 > lo ? s0 : lo) + tid;
                // four loads before their adds (which the compiler may not move them across)
                for (; j + 3 * kThreads < (end < s0 + kCached ? end : s0 + kCached); j += 4 * kThreads) {
                    uint32_t u[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) u[q] = keys[j - s0 + q * kThreads];
#pragma unroll
                    for (int q = 0; q < 4; ++q) count(u[q]);
                }
                for (; j < end; j += kThreads) count(key_at(j));
                __syncthreads();
                // bins in descending order, four a thread
                const int at = kBins - 4 - 4 * tid;
                int4 c = *reinterpret_cast<const int4*>(hist + at);
                if (kSliced) {
                    // bins [owner * per, ..) join at rank `owner`; per = 2048 / ranks, ranks >= 2
                    const int per = kBins / ranks, owner = at / per, slot = pass * (kBins / 2) + at % per;
                    const uint32_t to = at_rank(joined + slot, owner);
                    add_cluster(to, c.x), add_cluster(to + 4, c.y), add_cluster(to + 8, c.z), add_cluster(to + 12, c.w);
                    cluster_sync();
                    c = ld_cluster4(to);
                }
                const int sum = c.x + c.y + c.z + c.w;
                int above = sum;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const int y = __shfl_up_sync(0xFFFFFFFFu, above, off);
                    if (lane >= off) above += y;
                }
                if (lane == 31) scan[warp] = above;
                __syncthreads();
                above -= sum;  // keys in higher bins than this thread's
#pragma unroll
                for (int w = 0; w < kWarps; ++w) above += w < warp ? scan[w] : 0;
                if (above < need && above + sum >= need) {
                    int d = 3, in = c.w;
                    if (above + in < need) above += in, d = 2, in = c.z;
                    if (above + in < need) above += in, d = 1, in = c.y;
                    if (above + in < need) above += in, d = 0, in = c.x;
                    found = make_int4(at + d, need - above, in, 0);
                }
                __syncthreads();
                cut = pass == 0 ? (uint32_t)found.x : (cut << width) | (uint32_t)found.x;
                level = need = found.y;
                if (found.y == found.z) break;  // the whole bin stays
            }
        }
        // keys that stay for sure, and keys on the level
        int nk = 0, nt = 0;
        each([&](int j, uint32_t key) {
            const uint32_t u = key >> shift;
            const bool in = j < w1, forced = j < lo || j >= hi;
            nk += in && (forced || u > cut);
            nt += in && !forced && u == cut;
        });
        nk = __reduce_add_sync(0xFFFFFFFFu, nk), nt = __reduce_add_sync(0xFFFFFFFFu, nt);
        if (lane == 0) wkeep[warp] = nk, wtie[warp] = nt;
        __syncthreads();
        int keep_before = 0, tie_before = 0;
        if (kSliced) {
            if (warp == 0) {
                const int x = __reduce_add_sync(0xFFFFFFFFu, lane < kWarps ? wkeep[lane] : 0);
                const int y = __reduce_add_sync(0xFFFFFFFFu, lane < kWarps ? wtie[lane] : 0);
                if (lane == 0) counts = make_int4(x, y, 0, 0);
            }
            cluster_sync();
            int4 x = make_int4(0, 0, 0, 0);
            if (lane < rank) x = ld_cluster4(at_rank(&counts, lane));
            keep_before = __reduce_add_sync(0xFFFFFFFFu, x.x), tie_before = __reduce_add_sync(0xFFFFFFFFu, x.y);
        }
        keep_before += __reduce_add_sync(0xFFFFFFFFu, lane < warp && lane < kWarps ? wkeep[lane] : 0);
        tie_before += __reduce_add_sync(0xFFFFFFFFu, lane < warp && lane < kWarps ? wtie[lane] : 0);
        each([&](int j, uint32_t key) {
            const uint32_t u = key >> shift;
            const bool in = j < w1, forced = j < lo || j >= hi;
            const bool keep = in && (forced || u > cut), tie = in && !forced && u == cut;
            const uint32_t below = (1u << lane) - 1, km = __ballot_sync(0xFFFFFFFFu, keep),
                           tm = __ballot_sync(0xFFFFFFFFu, tie);
            const int ties = tie_before + __popc(tm & below);
            const int slot = keep_before + __popc(km & below) + (ties < level ? ties : level);
            // a CTA that selects alone writes its own share
            if ((keep || (tie && ties < level)) && (kSliced || (slot >= m0 && slot < m1))) {
                ids[slot] = j;
                so[slot] = key_score(key);
            }
            keep_before += __popc(km);
            tie_before += __popc(tm);
        });
    } else {
        for (int m = m0 + tid; m < m1 && m < kept; m += kThreads) {
            ids[m] = m;
            so[m] = sc[m];
        }
    }
    for (int m = (m0 > kept ? m0 : kept) + tid; m < m1; m += kThreads) {
        ids[m] = -1;
        so[m] = 0.0f;
    }
    if (kSliced)
        cluster_sync();  // the ids of every CTA; and no CTA leaves while its counts are read
    else
        __syncthreads();
    if (a.copy) copy_rows(a, b, h, m0, m1);
}

// The copy alone, for rows whose selecting CTAs are too few to draw the memory's bandwidth: every
// CTA an equal share of a row's slots.
__global__ void __launch_bounds__(kThreads, 2) evict_copy_kernel(const EvictArgs a, int ranks) {
    const int rank = blockIdx.x % ranks, row = blockIdx.x / ranks;
    copy_rows(a, row / a.Hkv, row % a.Hkv, (int)((int64_t)a.capacity * rank / ranks),
              (int)((int64_t)a.capacity * (rank + 1) / ranks));
}

}  // namespace
}  // namespace lsa

using namespace lsa;

extern "C" {

int lsa_evict(const void* k, const void* v, int64_t row_bytes, const int64_t* strides, const float* scores,
              const int32_t* lengths, int64_t B, int64_t T, int64_t Hkv, int64_t budget, int64_t window, int64_t sink,
              int64_t capacity, void* k_out, void* v_out, float* scores_out, int32_t* lengths_out, int32_t* ids,
              cudaStream_t stream) {
    if (B < 0 || T < 0 || Hkv <= 0 || row_bytes <= 0 || row_bytes % 16 || row_bytes > 65536) return LSA_ERR_ARG;
    if (window < 0 || sink < 0 || budget < 0 || window > budget || sink > budget - window || capacity < budget)
        return LSA_ERR_ARG;
    if (T > INT32_MAX - (1 << 16) || capacity > INT32_MAX - (1 << 16) || strides == nullptr) return LSA_ERR_ARG;
    for (int i = 0; i < 6; ++i)
        if (strides[i] < 0 || strides[i] % 16) return LSA_ERR_ARG;
    if (B == 0) return LSA_OK;
    if (lengths == nullptr || lengths_out == nullptr) return LSA_ERR_ARG;
    if (T > 0 && (k == nullptr || v == nullptr || scores == nullptr)) return LSA_ERR_ARG;
    if (capacity > 0 && (k_out == nullptr || v_out == nullptr || scores_out == nullptr || ids == nullptr))
        return LSA_ERR_ARG;
    for (const void* p : {k, v, (const void*)k_out, (const void*)v_out})
        if ((uintptr_t)p & 15) return LSA_ERR_ARG;
    if (B > INT32_MAX / 16 / Hkv) return LSA_ERR_SIZE;  // one cluster of at most 16 CTAs a row
    EvictArgs a;
    a.k = k, a.v = v;
    a.k_b = strides[0], a.k_t = strides[1], a.k_h = strides[2];
    a.v_b = strides[3], a.v_t = strides[4], a.v_h = strides[5];
    a.scores = scores, a.lengths = lengths;
    a.B = (int)B, a.T = (int)T, a.Hkv = (int)Hkv, a.row_bytes = (int)row_bytes;
    a.budget = (int)(budget < INT32_MAX ? budget : INT32_MAX), a.window = (int)window, a.sink = (int)sink;
    a.capacity = (int)capacity;
    a.k_out = k_out, a.v_out = v_out, a.scores_out = scores_out, a.lengths_out = lengths_out, a.ids = ids;
    a.row_lanes = row_bytes / 16 >= 32 ? 32 : next_pow2((int)(row_bytes / 16));
    // A row's CTAs. Keys that fit one CTA are selected by each of them: as many as have 64 slots to copy,
    // up to 128 in all (more than one an SM slow each other's selection: 9.6 us for a step of 8 rows in
    // 128 CTAs, 12.4 in 256), a second one for a large batch. More keys go in slices to a cluster of 8
    // (of 16 for few rows, or slices past its shared memory; it fills most of a GPC: 101 against 76
    // us for 32 rows of 131072 keys).
    const int64_t units = B * Hkv;
    const bool sliced = T > kCached;
    int64_t ranks = 1;
    while (units * ranks * 2 <= 148 && capacity / (2 * ranks) >= 64) ranks *= 2;
    if (units > 148 && units < 4 * 148) ranks = 2;
    if (sliced) ranks = units * 8 < 148 || T > 8 * kCached ? 16 : 8;
    const int64_t slice = sliced ? (T + ranks - 1) / ranks : T;
    const int smem = (int)((slice < kCached ? slice : kCached) * 4);
    auto kern = sliced ? evict_kernel<true> : evict_kernel<false>;
    if (!(sliced ? allow_kernel<evict_kernel<true>>(kCached * 4, true) : allow_kernel<evict_kernel<false>>(kCached * 4)))
        return LSA_ERR_CUDA;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = sliced ? (unsigned)ranks : 1;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    // few CTAs with much to copy leave it to a launch of its own
    a.copy = units * ranks >= 100 || units * capacity * row_bytes <= 4 << 20;
    if (cudaLaunchKernelEx(&cfg, kern, a, (int)ranks) != cudaSuccess) return LSA_ERR_CUDA;
    if (!a.copy) {
        const int64_t each = (4 * 148 + units - 1) / units;
        evict_copy_kernel<<<(unsigned)(units * each), kThreads, 0, stream>>>(a, (int)each);
        LSA_LAUNCH_CHECK();
    }
    return LSA_OK;
}

}  // extern "C"
