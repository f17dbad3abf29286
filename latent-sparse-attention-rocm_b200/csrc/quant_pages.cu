// quant_pages.cu - what writes the 8-bit paged cache: the append of new tokens, copies of pages (sm_100a).
//
// Append. A page's scale is the smallest power of two that holds the new tokens' largest magnitude, or the one
// it has where older tokens stay on the page and need more; older codes follow a scale that grows. A power of
// two, so that growing moves e4m3's exponents and changes no other bit above its smallest step, and an integer's
// successive roundings stay within one step of its scale. One CTA (or warp) a (sequence, page, KV head, K or V):
// the new rows stay in registers, as they lie in memory, between the maximum and the codes, so every byte moves once.
// Measured (B200, 8 heads, D 128, bf16 to e4m3, pages of 64): 4 x 16383 tokens, 403 MB, 63-68 us = 5.9-6.4 TB/s, 92-99 %
// of the measured copy rate. What counts is how many CTAs have rows in flight while others look their page up, reduce
// or store: 128 threads with eight rows of 16 bytes each; 256 threads with four 75 us, K and V in one CTA 95, registers
// bounded for more CTAs (spills) 89. 64 tokens: 2.0-2.4 us as graph replays, 7 to 10 in a loop (the host). Pages of 16
// tokens 96 us, 32 74, 128 70; int8 74; fp32, 2 x 16383 tokens, 336 MB, 55.
#include <type_traits>

#include "quant.cuh"

namespace lsa {
namespace {

// Largest magnitude of a lane's values (NaN counts as nothing), two at a time where they are 16 bits wide.
template <typename T, int N, typename Raw> __device__ __forceinline__ float largest(const Raw (&raw)[N]) {
    if constexpr (sizeof(T) == 2) {
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        T2 top;
#pragma unroll
        for (int i = 0; i < 4 * N; ++i) {
            const uint4& u = raw[i / 4].u[0];
            const uint32_t w = (i % 4 == 0 ? u.x : (i % 4 == 1 ? u.y : (i % 4 == 2 ? u.z : u.w))) & 0x7FFF7FFFu;
            top = i == 0 ? *reinterpret_cast<const T2*>(&w) : __hmax2(top, *reinterpret_cast<const T2*>(&w));
        }
        return fmaxf(to_f32(top.x), to_f32(top.y));
    } else {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float x[8];
            raw[i].floats(x);
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
        }
        return top;
    }
}

struct AppendArgs {
    const void *k, *v;
    int64_t k_b, k_t, k_h, v_b, v_t, v_h;
    uint8_t *k8, *v8;
    float *ks, *vs;
    const int32_t* table;
    int64_t table_ld;
    int M, pages, shift;
    const int32_t *lengths, *counts;  // counts: the rows of a sequence that are tokens, its last; null: all
    int B, Tq;
    uint32_t Hkv, units;  // units of a sequence: pages that its new tokens touch at most x heads x 2
};

constexpr int kSmallRows = 4;  // new tokens of a sequence that one warp takes

// Eight values as they lie in memory: half the registers of fp32, so more CTAs an SM have their rows in flight.
template <typename T> struct Raw {
    uint4 u[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const { load8<T>(reinterpret_cast<const T*>(u), x); }
};

// NT: threads of a (sequence, page, head, K or V); PASSES: of its rows.
template <typename T, int CODE, int D, int NT, int PASSES>
__global__ void __launch_bounds__(NT == 32 ? 128 : NT) append_kernel(const AppendArgs a) {
    constexpr int L = D / 8, RP = NT / L;  // lanes of a row, rows of a pass
    __shared__ float warp_top[NT / 32];
    const int tid = NT == 32 ? threadIdx.x & 31 : threadIdx.x;
    grid_wait();
    grid_trigger();
    // (pages x heads x K and V, sequences); 32-bit divisions: those of 64 bits took half of the kernel's time
    const uint32_t unit = NT == 32 ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (unit >= a.units) return;
    const bool value = unit & 1;
    const uint32_t nth = (unit >> 1) / a.Hkv;  // page of the call's
    const int h = (int)((unit >> 1) - nth * a.Hkv), b = blockIdx.y;
    const int64_t length = a.lengths[b];
    const int64_t start = length - a.Tq;         // position of the call's first row; negative: rows that are padding
    int64_t first = start < 0 ? 0 : start;
    if (a.counts) {
        const int count = a.counts[b];
        const int64_t from = length - (count < 0 ? 0 : (count > a.Tq ? a.Tq : count));
        first = first > from ? first : from;
    }
    const int64_t slot = (first >> a.shift) + nth;
    const int64_t p0 = slot << a.shift;
    const int page = 1 << a.shift;
    if (slot >= a.M || p0 >= length) return;
    const int id = a.table[b * a.table_ld + slot];
    if (id < 0 || id >= a.pages) return;
    const int kept = first > p0 ? (int)(first - p0) : 0;  // older tokens of the page
    const int end = length - p0 < page ? (int)(length - p0) : page;
    const int n = end - kept;
    if (n <= 0) return;  // a count of 0 in the middle of a page: no new token, nothing of the page changes
    const T* src = static_cast<const T*>(value ? a.v : a.k) + (value ? b * a.v_b + h * a.v_h : b * a.k_b + h * a.k_h);
    const int64_t ld = value ? a.v_t : a.k_t;
    const int64_t head = (int64_t)id * a.Hkv + h;
    uint8_t* dst = (value ? a.v8 : a.k8) + head * page * D;
    float* scale = (value ? a.vs : a.ks) + head;
    const int r = tid / L, c = tid % L * 8;
    src += (p0 + kept - start + r) * ld + c;

    float was = 0.0f;
    if (kept > 0) was = *scale;
    Raw<T> raw[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        raw[i].zero();
        if (i * RP + r < n) raw[i].load(src + (int64_t)i * RP * ld);
    }
    float top = fmaxf(0.0f, largest<T>(raw));
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, off));
    was = __shfl_sync(0xFFFFFFFFu, was, 0);  // every lane's read is behind it, before the write below
    if (NT > 32) {
        if ((tid & 31) == 0) warp_top[tid >> 5] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NT / 32; ++i) top = fmaxf(top, warp_top[i]);
    }
    const float needed = scale_for<CODE>(top);
    const float now = kept > 0 ? fmaxf(was, needed) : needed;
    if (tid == 0 && (kept == 0 || now != was)) *scale = now;
    // a scale of the caller's own need not be a power of two: then a division, as the codes are defined
    const bool power = (__float_as_uint(now) & 0x7FFFFFu) == 0;
    const float inv = power ? 1.0f / now : 1.0f;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        if (i * RP + r >= n) continue;
        float x[8];
        raw[i].floats(x);
        if (power) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= inv;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __fdiv_rn(x[e], now);
        }
        *reinterpret_cast<uint2*>(dst + (kept + i * RP + r) * D + c) =
            make_uint2(codes_of<CODE>(x[0], x[1], x[2], x[3]), codes_of<CODE>(x[4], x[5], x[6], x[7]));
    }
    if (kept > 0 && now != was) {  // now is a power of two
        for (int row = r; row < kept; row += RP) {
            uint2* at = reinterpret_cast<uint2*>(dst + row * D + c);
            const uint2 old = *at;
            float y[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t u = halves_of<CODE>(e < 2 ? old.x : old.y, e & 1);
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
                y[2 * e] = f.x * was * inv;
                y[2 * e + 1] = f.y * was * inv;
            }
            *at = make_uint2(codes_of<CODE>(y[0], y[1], y[2], y[3]), codes_of<CODE>(y[4], y[5], y[6], y[7]));
        }
    }
}

template <typename T, int CODE, int D> int launch(const AppendArgs& a, cudaStream_t stream) {
    if (a.Tq <= kSmallRows) {
        const dim3 blocks((a.units + 3) / 4, (unsigned)a.B);
        return launch_after(append_kernel<T, CODE, D, 32, kSmallRows * (D / 8) / 32>, blocks, 128, 0, stream, a);
    }
    constexpr int NT = D;  // 8 rows a pass (4 x 16k tokens, D 128: 128 threads 63 us, 256 75, 512 107)
    const dim3 grid(a.units, (unsigned)a.B);
    switch (a.shift) {
        case 4: return launch_after(append_kernel<T, CODE, D, NT, 2>, grid, NT, 0, stream, a);
        case 5: return launch_after(append_kernel<T, CODE, D, NT, 4>, grid, NT, 0, stream, a);
        case 6: return launch_after(append_kernel<T, CODE, D, NT, 8>, grid, NT, 0, stream, a);
        default: return launch_after(append_kernel<T, CODE, D, NT, 16>, grid, NT, 0, stream, a);
    }
}
template <typename T> int launch(const AppendArgs& a, int code, int64_t D, cudaStream_t stream) {
    if (code == kE4M3) return D == 64 ? launch<T, kE4M3, 64>(a, stream) : launch<T, kE4M3, 128>(a, stream);
    return D == 64 ? launch<T, kInt8, 64>(a, stream) : launch<T, kInt8, 128>(a, stream);
}

// Copies of pages: a CTA takes kCopy bytes of one pair's K or V.
constexpr int kCopyThreads = 256, kCopyDepth = 8;
constexpr int kCopy = kCopyThreads * kCopyDepth * 16;

__global__ void __launch_bounds__(kCopyThreads)
    move_pages_kernel(uint8_t* k8, uint8_t* v8, float* ks, float* vs, const int32_t* src, const int32_t* dst,
                      int64_t bytes, int Hkv, int pages, int chunks) {
    grid_wait();
    grid_trigger();
    const int64_t pair = blockIdx.x / (2 * chunks);
    const int part = (int)(blockIdx.x % (2 * chunks));
    const int s = src[pair], d = dst[pair];
    if (s < 0 || s >= pages || d < 0 || d >= pages || s == d) return;
    const bool value = part >= chunks;
    const int chunk = value ? part - chunks : part;
    uint8_t* base = value ? v8 : k8;
    const uint4* from = reinterpret_cast<const uint4*>(base + s * bytes);
    uint4* to = reinterpret_cast<uint4*>(base + d * bytes);
    const int64_t n = bytes / 16, i0 = (int64_t)chunk * (kCopy / 16) + threadIdx.x;
    uint4 u[kCopyDepth];
#pragma unroll
    for (int i = 0; i < kCopyDepth; ++i)
        if (i0 + i * kCopyThreads < n) u[i] = from[i0 + i * kCopyThreads];
    if (chunk == 0) {
        float* sc = value ? vs : ks;
        for (int h = threadIdx.x; h < Hkv; h += kCopyThreads) sc[(int64_t)d * Hkv + h] = sc[(int64_t)s * Hkv + h];
    }
#pragma unroll
    for (int i = 0; i < kCopyDepth; ++i)
        if (i0 + i * kCopyThreads < n) to[i0 + i * kCopyThreads] = u[i];
}

bool pool_ok(int code, int64_t pages, int64_t page, int64_t Hkv, int64_t D) {
    if (code != kE4M3 && code != kInt8) return false;
    if (pages < 0 || Hkv < 1 || (page != 16 && page != 32 && page != 64 && page != 128)) return false;
    return D == 64 || D == 128;
}

}  // namespace
}  // namespace lsa

extern "C" {

int lsa_append_quantized(const void* k, const void* v, int dtype, const int64_t* strides, void* k8, void* v8,
                         float* k_scale, float* v_scale, int code, int64_t pages, int64_t page, const int32_t* table,
                         int64_t table_ld, int64_t M, const int32_t* lengths, const int32_t* counts, int64_t B,
                         int64_t Tq, int64_t Hkv, int64_t D, cudaStream_t stream) {
    using namespace lsa;
    if (!pool_ok(code, pages, page, Hkv, D) || dtype < 0 || dtype > 2 || strides == nullptr) return LSA_ERR_ARG;
    if (B < 0 || Tq < 0 || M < 0) return LSA_ERR_ARG;
    if (B == 0 || Tq == 0 || M == 0 || pages == 0) return LSA_OK;
    if (!k || !v || !k8 || !v8 || !k_scale || !v_scale || !table || !lengths) return LSA_ERR_ARG;
    const int64_t unit = 16 / (dtype == kF32 ? 4 : 2);
    for (int i = 0; i < 6; ++i)
        if (strides[i] < 0 || strides[i] % unit != 0) return LSA_ERR_ARG;
    for (const void* p : {k, v, (const void*)k8, (const void*)v8})
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return LSA_ERR_ARG;
    if (pages > INT32_MAX || M > INT32_MAX || B > INT32_MAX || Tq > INT32_MAX || Hkv > 65535) return LSA_ERR_SIZE;
    AppendArgs a = {};
    a.k = k, a.v = v;
    a.k_b = strides[0], a.k_t = strides[1], a.k_h = strides[2];
    a.v_b = strides[3], a.v_t = strides[4], a.v_h = strides[5];
    a.k8 = static_cast<uint8_t*>(k8), a.v8 = static_cast<uint8_t*>(v8);
    a.ks = k_scale, a.vs = v_scale;
    a.table = table, a.table_ld = table_ld, a.M = (int)M, a.pages = (int)pages;
    a.shift = page == 16 ? 4 : (page == 32 ? 5 : (page == 64 ? 6 : 7));
    a.lengths = lengths, a.counts = counts;
    a.B = (int)B, a.Tq = (int)Tq, a.Hkv = (uint32_t)Hkv;
    const int64_t slots = (Tq + page - 2) / page + 1;
    const int64_t units = (slots < M ? slots : M) * Hkv * 2;
    if (B > 65535 || units > INT32_MAX) return LSA_ERR_SIZE;
    a.units = (uint32_t)units;
    switch (dtype) {
        case kF32: return launch<float>(a, code, D, stream);
        case kF16: return launch<__half>(a, code, D, stream);
        default: return launch<__nv_bfloat16>(a, code, D, stream);
    }
}

int lsa_move_pages(void* k8, void* v8, float* k_scale, float* v_scale, int64_t pages, int64_t page, int64_t Hkv,
                   int64_t D, const int32_t* src, const int32_t* dst, int64_t n, cudaStream_t stream) {
    using namespace lsa;
    if (!pool_ok(kE4M3, pages, page, Hkv, D) || n < 0) return LSA_ERR_ARG;
    if (n == 0 || pages == 0) return LSA_OK;
    if (!k8 || !v8 || !k_scale || !v_scale || !src || !dst) return LSA_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(k8) % 16 != 0 || reinterpret_cast<uintptr_t>(v8) % 16 != 0) return LSA_ERR_ARG;
    if (pages > INT32_MAX || Hkv > 65535) return LSA_ERR_SIZE;
    const int64_t bytes = Hkv * page * D, chunks = (bytes + kCopy - 1) / kCopy;
    if (n > INT32_MAX / (2 * chunks)) return LSA_ERR_SIZE;
    return launch_after(move_pages_kernel, dim3((unsigned)(n * 2 * chunks)), kCopyThreads, 0, stream,
                        static_cast<uint8_t*>(k8), static_cast<uint8_t*>(v8), k_scale, v_scale, src, dst, bytes,
                        (int)Hkv, (int)pages, (int)chunks);
}

}  // extern "C"
