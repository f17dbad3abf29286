// rotate.cu - norms of queries and keys for each head, with the position rotation, in one pass (sm_100a).
//
// For a head's D values x of a token at position p:
//   y = x * rsqrt(mean(x^2) + eps) * w                      (where a weight is given)
//   (a, b) -> amplitude * (a cos t - b sin t, a sin t + b cos t),  t = p f_i,  i < R / 2
// over the pairs (y_i, y_{i + R/2}) or, interleaved, (y_2i, y_2i+1); the values past R are not rotated. All in
// fp32, rounded once. The angle in turns is p * (f / 2 pi) in fp64, reduced there to half a turn either way
// (off by 2^-27 of a turn at most below position 2^26) and then rounded to fp32.
//
// A warp holds a token's heads one after another, D / 8 lanes a head, and its lanes' angles once for all of them. A
// lane has four values of either half and so both of a pair, in the half layout as in the interleaved one (two
// 8-byte loads where one of 16 would want its partner's values by shuffle: 213 us became 138 with the packed
// arithmetic). A token's heads go to several warps where the tokens alone would not fill the SMs.
// Measured (B200, 32 + 8 heads, D 128, bf16, norms): 2 x 16384 tokens, 671 MB, 112-121 us = 5.5-6.0 TB/s, 86-93 % of the measured
// copy rate; bounded by issue and the loads' latency together: 80 registers leave 24 warps an SM, and bounding them to 64
// spills (158 us). 64 tokens: 2.6 us as graph replays, 9 to 13 called in a loop (the host). fp32, 2 x 8192 tokens, the same
// bytes: 130 us; D 64 62 us (335 MB), D 256 231 (1342 MB); interleaved, or half of a head turned, 120.
#include "pairs.cuh"

namespace lsa {
namespace {

constexpr int kWarps = 4;
constexpr int kAhead = 3;  // rows a lane group has in flight (2 x 16k tokens: 2 120 us, 3 111, 4 122, 6 118, 8 127)

struct RotateArgs {
    const void *q, *k;
    int64_t q_b, q_t, q_h, k_b, k_t, k_h;
    const void* positions;
    int64_t pos_b, pos_t;
    const double* frequencies;
    const void *q_weight, *k_weight;
    void *q_out, *k_out;
    int64_t tokens;
    int T, Hq, Hkv, R, sections;
    int wide_positions, q_weight_f32, k_weight_f32;
    float amplitude, eps;
};

// Eight values of a lane, four at either of two places, as they lie in memory.
template <typename T> struct Raw8 {
    uint2 u[2];
    __device__ __forceinline__ void load(const T* p, int off) {
        u[0] = *reinterpret_cast<const uint2*>(p);
        u[1] = *reinterpret_cast<const uint2*>(p + off);
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const { load8<T>(reinterpret_cast<const T*>(u), x); }
};
template <> struct Raw8<float> {
    uint4 u[2];
    __device__ __forceinline__ void load(const float* p, int off) {
        u[0] = *reinterpret_cast<const uint4*>(p);
        u[1] = *reinterpret_cast<const uint4*>(p + off);
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const { load8<float>(reinterpret_cast<const float*>(u), x); }
};

__device__ __forceinline__ uint32_t two(float a, float b, __nv_bfloat16*) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t two(float a, float b, __half*) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T> __device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
    *reinterpret_cast<uint2*>(p) = make_uint2(two(a, b, (T*)nullptr), two(c, d, (T*)nullptr));
}
template <> __device__ __forceinline__ void store4<float>(float* p, float a, float b, float c, float d) {
    *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}

// Sine and cosine of a turn's fraction, |turn| <= 1/2. For values that are rounded to 16 bits the special-function
// unit's (2^-21 off at most on +-pi, and 2^-22 for the argument, against 2^-12 and 2^-9 of the rounding).
template <typename T> __device__ __forceinline__ void sin_cos(float turn, float* s, float* c) {
    const float x = turn * 6.283185307179586f;
    *s = __sinf(x), *c = __cosf(x);
}
template <> __device__ __forceinline__ void sin_cos<float>(float turn, float* s, float* c) {
    sincospif(turn + turn, s, c);
}

// WHOLE: all of a head turns (R = D).
template <typename T, int D, bool INTER, bool WHOLE>
__global__ void __launch_bounds__(kWarps * 32) norm_rotate_kernel(const RotateArgs a) {
    constexpr int L = D / 8;  // lanes of a head
    constexpr int N = 32 / L; // heads of a pass
    const int lane = threadIdx.x & 31, j = lane % L, own = lane / L;
    const int64_t unit = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    // (64-bit divisions only where the tokens want them)
    const int64_t token = a.sections == 1 ? unit : (int64_t)((uint32_t)unit / (uint32_t)a.sections);
    const int section = (int)(unit - token * a.sections);
    grid_wait();
    grid_trigger();
    if (token >= a.tokens) return;
    const int64_t b = a.tokens <= INT32_MAX ? (int64_t)((uint32_t)token / (uint32_t)a.T) : token / a.T, t = token - b * a.T;
    // passes over q's heads, then k's; this warp's
    const int q_passes = (a.Hq + N - 1) / N, passes = q_passes + (a.Hkv + N - 1) / N;
    const int p0 = passes * section / a.sections, p1 = passes * (section + 1) / a.sections;

    // the lane's values: four from `at0` on, four `step` further
    const bool turns = WHOLE || 8 * j < a.R;
    const int at0 = INTER || !turns ? 8 * j : 4 * j, step = INTER || !turns ? 4 : a.R / 2;
    const T* qrow = static_cast<const T*>(a.q) + b * a.q_b + t * a.q_t + own * a.q_h + at0;
    const T* krow = static_cast<const T*>(a.k) + b * a.k_b + t * a.k_t + own * a.k_h + at0;
    T* qdst = static_cast<T*>(a.q_out) + (token * a.Hq + own) * D + at0;
    T* kdst = static_cast<T*>(a.k_out) + (token * a.Hkv + own) * D + at0;
    // passes that this lane has a head in: the last of q's and of k's may be short of heads
    const int q_live = (a.Hq - own + N - 1) / N, k_live = q_passes + (a.Hkv - own + N - 1) / N;
    auto is_q = [&](int p) { return p < q_passes; };
    auto live = [&](int p) { return p < (is_q(p) ? q_live : k_live); };
    const bool from_q = is_q(p0);
    const T* src = from_q ? qrow + (int64_t)p0 * N * a.q_h : krow + (int64_t)(p0 - q_passes) * N * a.k_h;
    T* dst = from_q ? qdst + (int64_t)p0 * N * D : kdst + (int64_t)(p0 - q_passes) * N * D;
    const int64_t q_next = N * a.q_h, k_next = N * a.k_h;
    auto load = [&](Raw8<T>& raw, int p) {  // in the order of the passes
        if (p < p1 && live(p)) raw.load(src, step);
        src = p + 1 == q_passes ? krow : src + (is_q(p) ? q_next : k_next);
    };
    Raw8<T> raw[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load(raw[i], p0 + i);

    const int64_t at = b * a.pos_b + t * a.pos_t;
    const double position = a.wide_positions ? (double)static_cast<const int64_t*>(a.positions)[at]
                                             : (double)static_cast<const int32_t*>(a.positions)[at];
    float cs[4], sn[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        cs[i] = 1.0f, sn[i] = 0.0f;
        if (turns) {
            double turn = position * (a.frequencies[4 * j + i] * 0.15915494309189535);
            turn -= rint(turn);
            sin_cos<T>((float)turn, &sn[i], &cs[i]);
            cs[i] *= a.amplitude;
            sn[i] *= a.amplitude;
        }
    }
    // Pair e's new values are r (x_u uu - x_v vu) and r (x_v vv + x_u uv): the weights are in the rotation.
    float uu[4], vu[4], vv[4], uv[4];
    const void* weights = nullptr;
    auto take = [&](const void* src, int f32) {
        weights = src;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float wu = 1.0f, wv = 1.0f;
            if (src) {
                const int u = INTER ? 2 * e : e, v = INTER ? 2 * e + 1 : e + 4;
                const int iu = at0 + (u < 4 ? u : step + u - 4), iv = at0 + (v < 4 ? v : step + v - 4);
                wu = f32 ? static_cast<const float*>(src)[iu] : to_f32(static_cast<const T*>(src)[iu]);
                wv = f32 ? static_cast<const float*>(src)[iv] : to_f32(static_cast<const T*>(src)[iv]);
            }
            uu[e] = wu * cs[e], vu[e] = wv * sn[e], vv[e] = wv * cs[e], uv[e] = wu * sn[e];
        }
    };
    if (is_q(p0)) take(a.q_weight, a.q_weight_f32);
    bool on_k = false;

    for (int base = p0; base < p1; base += kAhead) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int p = base + i;
            if (p >= p1) break;
            if (!is_q(p) && !on_k) {
                on_k = true;
                take(a.k_weight, a.k_weight_f32);
            }
            float x[8];
            raw[i].floats(x);
            load(raw[i], p + kAhead);
            float r = 1.0f;
            if (weights) {
                uint64_t two = mul2(pair(x[0], x[1]), pair(x[0], x[1]));
#pragma unroll
                for (int e = 2; e < 8; e += 2) two = fma2(pair(x[e], x[e + 1]), pair(x[e], x[e + 1]), two);
                float s0, s1;
                unpair(two, s0, s1);
                float sum = s0 + s1;
#pragma unroll
                for (int off = L / 2; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
                r = rsqrtf(sum * (1.0f / D) + a.eps);
            }
            const uint64_t rr = pair(r, r);
            float y[8];
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const int u0 = INTER ? 2 * e : e, u1 = INTER ? 2 * e + 2 : e + 1, dv = INTER ? 1 : 4;
                const uint64_t xu = mul2(pair(x[u0], x[u1]), rr), xv = mul2(pair(x[u0 + dv], x[u1 + dv]), rr);
                unpair(fma2(xu, pair(uu[e], uu[e + 1]), mul2(xv, pair(-vu[e], -vu[e + 1]))), y[u0], y[u1]);
                unpair(fma2(xv, pair(vv[e], vv[e + 1]), mul2(xu, pair(uv[e], uv[e + 1]))), y[u0 + dv], y[u1 + dv]);
                // an infinity that does not turn stays its own: times a sine of 0 it would be a NaN of its neighbour's (WHOLE keeps the test
                // out where there is nothing to test: 111 us against 120)
                if (!WHOLE && !turns) {
                    unpair(mul2(xu, pair(uu[e], uu[e + 1])), y[u0], y[u1]);
                    unpair(mul2(xv, pair(vv[e], vv[e + 1])), y[u0 + dv], y[u1 + dv]);
                }
            }
            if (live(p)) {
                store4<T>(dst, y[0], y[1], y[2], y[3]);
                store4<T>(dst + step, y[4], y[5], y[6], y[7]);
            }
            dst = p + 1 == q_passes ? kdst : dst + N * D;
        }
    }
}

template <typename T, int D, bool INTER> int launch(const RotateArgs& a, unsigned grid, cudaStream_t stream) {
    return a.R == D ? launch_after(norm_rotate_kernel<T, D, INTER, true>, dim3(grid), kWarps * 32, 0, stream, a)
                    : launch_after(norm_rotate_kernel<T, D, INTER, false>, dim3(grid), kWarps * 32, 0, stream, a);
}
template <typename T, int D> int launch(const RotateArgs& a, bool inter, unsigned grid, cudaStream_t stream) {
    return inter ? launch<T, D, true>(a, grid, stream) : launch<T, D, false>(a, grid, stream);
}
template <typename T> int launch(const RotateArgs& a, int64_t D, bool inter, unsigned grid, cudaStream_t stream) {
    return D == 64 ? launch<T, 64>(a, inter, grid, stream)
                   : (D == 128 ? launch<T, 128>(a, inter, grid, stream) : launch<T, 256>(a, inter, grid, stream));
}

}  // namespace
}  // namespace lsa

extern "C" int lsa_norm_rotate(const void* q, const void* k, int dtype, const int64_t* strides, int64_t B, int64_t T,
                               int64_t Hq, int64_t Hkv, int64_t D, const void* positions, int wide_positions,
                               int64_t pos_b, int64_t pos_t, const double* frequencies, int64_t R, int interleaved,
                               float amplitude, const void* q_weight, int q_weight_dtype, const void* k_weight,
                               int k_weight_dtype, float eps, void* q_out, void* k_out, cudaStream_t stream) {
    using namespace lsa;
    if (strides == nullptr || B < 0 || T < 0 || Hq < 1 || Hkv < 1 || dtype < 0 || dtype > 2) return LSA_ERR_ARG;
    if ((D != 64 && D != 128 && D != 256) || R < 0 || R > D || R % 16 != 0) return LSA_ERR_ARG;
    if ((q_weight && q_weight_dtype != dtype && q_weight_dtype != kF32) ||
        (k_weight && k_weight_dtype != dtype && k_weight_dtype != kF32))
        return LSA_ERR_ARG;
    if (B == 0 || T == 0) return LSA_OK;
    if (!q || !k || !positions || (R > 0 && !frequencies) || !q_out || !k_out) return LSA_ERR_ARG;
    const int64_t unit = 16 / (dtype == kF32 ? 4 : 2);
    for (int i = 0; i < 6; ++i)
        if (strides[i] < 0 || strides[i] % unit != 0) return LSA_ERR_ARG;
    for (const void* p : {q, k, (const void*)q_out, (const void*)k_out, q_weight, k_weight})
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return LSA_ERR_ARG;
    if (T > INT32_MAX || Hq + Hkv > 65536 || B > INT64_MAX / (T * 65536)) return LSA_ERR_SIZE;
    RotateArgs a = {};
    a.q = q, a.k = k;
    a.q_b = strides[0], a.q_t = strides[1], a.q_h = strides[2];
    a.k_b = strides[3], a.k_t = strides[4], a.k_h = strides[5];
    a.positions = positions, a.wide_positions = wide_positions, a.pos_b = pos_b, a.pos_t = pos_t;
    a.frequencies = frequencies;
    a.q_weight = q_weight, a.k_weight = k_weight;
    a.q_weight_f32 = q_weight_dtype == kF32, a.k_weight_f32 = k_weight_dtype == kF32;
    a.q_out = q_out, a.k_out = k_out;
    a.tokens = B * T, a.T = (int)T, a.Hq = (int)Hq, a.Hkv = (int)Hkv, a.R = (int)R;
    a.amplitude = amplitude, a.eps = eps;
    // a token's heads over several warps where the tokens alone would not fill the SMs
    const int64_t each = 256 / D, passes = (Hq + each - 1) / each + (Hkv + each - 1) / each;
    int64_t sections = (148 * 16 + a.tokens - 1) / a.tokens;
    a.sections = (int)(sections < 1 ? 1 : (sections > passes ? passes : sections));
    const int64_t blocks = (a.tokens * a.sections + kWarps - 1) / kWarps;
    if (blocks > INT32_MAX) return LSA_ERR_SIZE;
    const bool inter = interleaved != 0;
    switch (dtype) {
        case kF32: return launch<float>(a, D, inter, (unsigned)blocks, stream);
        case kF16: return launch<__half>(a, D, inter, (unsigned)blocks, stream);
        default: return launch<__nv_bfloat16>(a, D, inter, (unsigned)blocks, stream);
    }
}
