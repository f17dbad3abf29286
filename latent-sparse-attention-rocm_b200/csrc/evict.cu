// evict.cu - eviction from a KV cache by accumulated attention weight (sm_100a).
//
// For sequence b with n keys and KV head h: n <= budget keeps every key; else the sinks
// [0, sink), the window [n - window, n) and, of the keys between, the budget - sink - window
// with the highest score stay. Scores order as the selection's packed keys do (ordered_bits:
// -NaN < -inf < ... < -0 < +0 < ... < +inf < +NaN), ties go to the lower index. The kept keys
// keep their order: out slot m holds kept key ids[m], ascending; slots past the kept count are
// zeros (ids -1).
#include "common.cuh"

namespace lsa {
namespace {

constexpr int kSelThreads = 1024;

struct EvictArgs {
    const void *k, *v;
    int64_t k_b, k_t, k_h, v_b, v_t, v_h;  // strides in bytes
    const float* scores;                   // [B, Hkv, T]
    const int32_t* lengths;                // [B]
    int B, T, Hkv, row_bytes;
    int budget, window, sink, capacity;
    void *k_out, *v_out;                   // [B, capacity, Hkv, D] contiguous
    float* scores_out;                     // [B, Hkv, capacity]
    int32_t* lengths_out;                  // [B]
    int32_t* ids;                          // [B, Hkv, capacity]
};

__device__ __forceinline__ uint32_t score_key(float f) { return (uint32_t)ordered_bits(f) ^ 0x80000000u; }

// One CTA per (sequence, KV head): the key of the last score that stays by a radix search
// (8 bits a pass, highest first), then an ordered compaction.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictArgs a) {
    __shared__ int hist[256], scan_sm[40], s_digit, s_need;
    const int h = blockIdx.x % a.Hkv, b = blockIdx.x / a.Hkv, tid = threadIdx.x;
    int n = a.lengths[b];
    n = n < 0 ? 0 : (n > a.T ? a.T : n);
    const int kept = n < a.budget ? n : a.budget;
    const float* sc = a.scores + ((int64_t)b * a.Hkv + h) * a.T;
    int32_t* ids = a.ids + ((int64_t)b * a.Hkv + h) * a.capacity;
    float* so = a.scores_out + ((int64_t)b * a.Hkv + h) * a.capacity;
    if (h == 0 && tid == 0) a.lengths_out[b] = kept;
    const int lo = a.sink, hi = n - a.window;  // the keys that compete, when n > budget
    uint32_t cut = 0;
    int level = 0;  // keys equal to the cut that stay
    if (n > a.budget) {
        int need = a.budget - a.sink - a.window;
        if (need == 0) {
            cut = 0xFFFFFFFFu;  // nothing is above it, and none of the level stays
        } else {
            for (int shift = 24; shift >= 0; shift -= 8) {
                for (int i = tid; i < 256; i += kSelThreads) hist[i] = 0;
                __syncthreads();
                for (int j = lo + tid; j < hi; j += kSelThreads) {
                    const uint32_t u = score_key(sc[j]);
                    if (shift == 24 || (u >> (shift + 8)) == (cut >> (shift + 8))) atomicAdd(&hist[(u >> shift) & 255], 1);
                }
                __syncthreads();
                if (tid == 0) {
                    int d = 255, above = 0;
                    while (above + hist[d] < need) above += hist[d--];
                    s_digit = d;
                    s_need = need - above;
                }
                __syncthreads();
                cut |= (uint32_t)s_digit << shift;
                need = s_need;
            }
            level = need;
        }
    }
    int out = 0, taken = 0;  // kept keys and level keys before this chunk
    for (int j0 = 0; j0 < n; j0 += kSelThreads) {
        const int j = j0 + tid;
        bool stay = false, tie = false;
        if (j < n) {
            if (n <= a.budget || j < lo || j >= hi) {
                stay = true;
            } else {
                const uint32_t u = score_key(sc[j]);
                stay = u > cut;
                tie = u == cut;
            }
        }
        int total;
        const int ties_before = taken + block_exclusive_scan(tie, scan_sm, &total);
        taken += total;
        if (tie && ties_before < level) stay = true;
        const int at = out + block_exclusive_scan(stay, scan_sm, &total);
        out += total;
        if (stay) {
            ids[at] = j;
            so[at] = sc[j];
        }
    }
    for (int m = kept + tid; m < a.capacity; m += kSelThreads) {
        ids[m] = -1;
        so[m] = 0.0f;
    }
}

// Rows of K and V by the kept ids, 16 bytes a thread; zeros past the kept count.
__global__ void __launch_bounds__(256) evict_gather_kernel(const EvictArgs a) {
    const int chunks = a.row_bytes / 16;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int c = (int)(i % chunks);
    const int64_t m = i / chunks;
    if (m >= a.capacity) return;
    const int h = blockIdx.y, b = blockIdx.z;
    const int id = a.ids[((int64_t)b * a.Hkv + h) * a.capacity + m];
    uint4 x = make_uint4(0, 0, 0, 0), y = x;
    if (id >= 0) {
        x = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.k) + b * a.k_b + id * a.k_t + h * a.k_h + c * 16);
        y = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.v) + b * a.v_b + id * a.v_t + h * a.v_h + c * 16);
    }
    const int64_t to = (((int64_t)b * a.capacity + m) * a.Hkv + h) * a.row_bytes + c * 16;
    *reinterpret_cast<uint4*>(static_cast<uint8_t*>(a.k_out) + to) = x;
    *reinterpret_cast<uint4*>(static_cast<uint8_t*>(a.v_out) + to) = y;
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
    if (T > INT32_MAX - 4096 || capacity > INT32_MAX - 4096 || strides == nullptr) return LSA_ERR_ARG;
    for (int i = 0; i < 6; ++i)
        if (strides[i] < 0 || strides[i] % 16) return LSA_ERR_ARG;
    if (B == 0) return LSA_OK;
    if (lengths == nullptr || lengths_out == nullptr) return LSA_ERR_ARG;
    if (T > 0 && (k == nullptr || v == nullptr || scores == nullptr)) return LSA_ERR_ARG;
    if (capacity > 0 && (k_out == nullptr || v_out == nullptr || scores_out == nullptr || ids == nullptr))
        return LSA_ERR_ARG;
    for (const void* p : {k, v, (const void*)k_out, (const void*)v_out})
        if ((uintptr_t)p & 15) return LSA_ERR_ARG;
    if (B > 65535 || Hkv > 65535 || B * Hkv > INT32_MAX) return LSA_ERR_SIZE;
    EvictArgs a;
    a.k = k, a.v = v;
    a.k_b = strides[0], a.k_t = strides[1], a.k_h = strides[2];
    a.v_b = strides[3], a.v_t = strides[4], a.v_h = strides[5];
    a.scores = scores, a.lengths = lengths;
    a.B = (int)B, a.T = (int)T, a.Hkv = (int)Hkv, a.row_bytes = (int)row_bytes;
    a.budget = (int)(budget < INT32_MAX ? budget : INT32_MAX), a.window = (int)window, a.sink = (int)sink;
    a.capacity = (int)capacity;
    a.k_out = k_out, a.v_out = v_out, a.scores_out = scores_out, a.lengths_out = lengths_out, a.ids = ids;
    evict_select_kernel<<<(unsigned)(B * Hkv), kSelThreads, 0, stream>>>(a);
    LSA_LAUNCH_CHECK();
    if (capacity > 0) {
        const int64_t work = capacity * (row_bytes / 16);
        dim3 grid((unsigned)((work + 255) / 256), (unsigned)Hkv, (unsigned)B);
        evict_gather_kernel<<<grid, 256, 0, stream>>>(a);
        LSA_LAUNCH_CHECK();
    }
    return LSA_OK;
}

}  // extern "C"
