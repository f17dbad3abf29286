// rotate.cu - norms of queries and keys for each head, with the position rotation, in one pass (sm_100a).
//
// For a head's D values x of a token at position p:
//   y = x * rsqrt(mean(x^2) + eps) * w                      (where a weight is given)
//   (a, b) -> amplitude * (a cos t - b sin t, a sin t + b cos t),  t = p f_i,  i < R / 2
// over the pairs (y_i, y_{i + R/2}) or, interleaved, (y_2i, y_2i+1); the values past R are not rotated. All in
// fp32, rounded once. The angle in turns is p * (f / 2 pi) in fp64, reduced there to half a turn either way:
// what is left of a position's 2^-53 is the angle's error, whatever the position.
//
// A warp holds a token's heads one after another, D / 8 lanes a head (8 values a lane), and its lanes' angles
// once for all of them; half-layout partners are a lane apart and change values by shuffle.
#include "launch.cuh"

namespace lsa {
namespace {

constexpr int kWarps = 4;
constexpr int kAhead = 4;  // rows a lane group has in flight

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

template <typename T> struct Raw8 {
    uint4 u;
    __device__ __forceinline__ void load(const T* p) { u = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void floats(float (&x)[8]) const { load8<T>(reinterpret_cast<const T*>(&u), x); }
};
template <> struct Raw8<float> {
    uint4 u[2];
    __device__ __forceinline__ void load(const float* p) {
        u[0] = reinterpret_cast<const uint4*>(p)[0];
        u[1] = reinterpret_cast<const uint4*>(p)[1];
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const { load8<float>(reinterpret_cast<const float*>(u), x); }
};

template <typename T> __device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    uint4 u;
    T* h = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = from_f32<T>(x[e]);
    *reinterpret_cast<uint4*>(p) = u;
}
template <> __device__ __forceinline__ void store8<float>(float* p, const float (&x)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

template <typename T, int D, bool INTER>
__global__ void __launch_bounds__(kWarps * 32) norm_rotate_kernel(const RotateArgs a) {
    constexpr int L = D / 8;    // lanes of a head
    constexpr int N = 32 / L;   // heads of a pass
    constexpr int A = INTER ? 4 : 8;
    const int lane = threadIdx.x & 31, j = lane % L;
    const int64_t unit = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int64_t token = unit / a.sections;
    const int section = (int)(unit - token * a.sections);
    grid_wait();
    grid_trigger();
    if (token >= a.tokens) return;
    const int64_t b = token / a.T, t = token - b * a.T;
    const int heads = a.Hq + a.Hkv;
    const int h0 = (int)((int64_t)heads * section / a.sections), h1 = (int)((int64_t)heads * (section + 1) / a.sections);

    const T* qrow = static_cast<const T*>(a.q) + b * a.q_b + t * a.q_t + j * 8;
    const T* krow = static_cast<const T*>(a.k) + b * a.k_b + t * a.k_t + j * 8;
    auto src = [&](int h) { return h < a.Hq ? qrow + h * a.q_h : krow + (h - a.Hq) * a.k_h; };
    Raw8<T> raw[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        const int h = h0 + i * N + lane / L;
        if (h < h1) raw[i].load(src(h));
    }

    const int64_t at = b * a.pos_b + t * a.pos_t;
    const double p = a.wide_positions ? (double)static_cast<const int64_t*>(a.positions)[at]
                                      : (double)static_cast<const int32_t*>(a.positions)[at];
    // half layout: a lane's 8 values lie in one half (R is a multiple of 16)
    const int half = a.R / 2;
    const bool turns = 8 * j < a.R, second = !INTER && 8 * j >= half;
    const int partner = INTER || !turns ? lane : (second ? lane - half / 8 : lane + half / 8);
    float cs[A], sn[A];
#pragma unroll
    for (int i = 0; i < A; ++i) {
        cs[i] = 1.0f, sn[i] = 0.0f;
        if (turns) {
            const int f = INTER ? 4 * j + i : 8 * j - (second ? half : 0) + i;
            double turn = p * (a.frequencies[f] * 0.15915494309189535);
            turn -= rint(turn);
            sincospif((float)(turn + turn), &sn[i], &cs[i]);
            cs[i] *= a.amplitude;
            sn[i] *= second ? a.amplitude : -a.amplitude;  // of the partner's value
        }
    }
    float w[8];
    bool norm = false;
    auto weight = [&](const void* src, int f32) {
        norm = src != nullptr;
        if (!norm) return;
        if (f32)
            load8<float>(static_cast<const float*>(src) + j * 8, w);
        else
            load8<T>(static_cast<const T*>(src) + j * 8, w);
    };
    int held = -1;  // whose weight w is: 0 q's, 1 k's

    for (int base = h0; base < h1; base += kAhead * N) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int h = base + i * N + lane / L;
            if (base + i * N >= h1) break;
            const bool live = h < h1;
            float x[8];
            if (live) {
                raw[i].floats(x);
                const int next = h + kAhead * N;
                if (next < h1) raw[i].load(src(next));
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = 0.0f;
            }
            const int whose = h < a.Hq ? 0 : 1;
            if (held != whose) {
                held = whose;
                weight(whose ? a.k_weight : a.q_weight, whose ? a.k_weight_f32 : a.q_weight_f32);
            }
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], sum);
#pragma unroll
            for (int off = L / 2; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
            if (norm) {
                const float r = rsqrtf(sum * (1.0f / D) + a.eps);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = x[e] * r * w[e];
            }
            float y[8];
            if (INTER) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {  // sn: minus the sine
                    y[2 * e] = fmaf(x[2 * e], cs[e], x[2 * e + 1] * sn[e]);
                    y[2 * e + 1] = fmaf(x[2 * e + 1], cs[e], -(x[2 * e] * sn[e]));
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float o = __shfl_sync(0xFFFFFFFFu, x[e], partner);
                    y[e] = fmaf(x[e], cs[e], o * sn[e]);
                }
            }
            if (live)
                store8<T>(h < a.Hq ? static_cast<T*>(a.q_out) + (token * a.Hq + h) * D + j * 8
                                   : static_cast<T*>(a.k_out) + (token * a.Hkv + h - a.Hq) * D + j * 8,
                          y);
        }
    }
}

template <typename T, int D> int launch(const RotateArgs& a, bool inter, unsigned grid, cudaStream_t stream) {
    return inter ? launch_after(norm_rotate_kernel<T, D, true>, dim3(grid), kWarps * 32, 0, stream, a)
                 : launch_after(norm_rotate_kernel<T, D, false>, dim3(grid), kWarps * 32, 0, stream, a);
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
        if (strides[i] % unit != 0) return LSA_ERR_ARG;
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
    const int64_t passes = (Hq + Hkv + 256 / D - 1) / (256 / D);
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
