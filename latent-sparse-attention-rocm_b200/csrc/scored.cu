// scored.cu - attention weights of the own keys of fp32 caches, added to a running score (sm_100a).
//
// With every row's lse known (prefix.cuh), key j of sequence b and KV head h gains
//   w_j = sum over the rows r = (token, head of the group) that see j of 2^(s_rj - lse_r)
// (log2 domain), the total attention it received. One thread owns a key, so the sum has one
// order and one writer: no atomics, the same bits every time. K is read a second time and nothing is in flight
// while a block computes: 8 caches of up to 8191 keys (32 / 8 heads, D 128) take 415 us with the attention, where
// the bytes take 62.
#include "prefix.cuh"

namespace lsa {
namespace {

constexpr int kWKeys = 128;  // keys of a CTA: one per thread
constexpr int kWRows = 8;    // query rows staged at a time

// fp32 inputs: the scores computed again on the FMA pipes, eight rows at a time.
template <int D>
__global__ void __launch_bounds__(kWKeys) own_weights_kernel(const PrefixArgs a, const float* __restrict__ scores,
                                                             float* __restrict__ scores_out) {
    constexpr int LDK = D + 4;
    extern __shared__ float sm[];
    float* sk = sm;                // [kWKeys][LDK]
    float* sq = sm + kWKeys * LDK; // [kWRows][D]
    __shared__ float slse[kWRows];
    const int per = (int)(((int64_t)a.T + kWKeys - 1) / kWKeys), bh = blockIdx.x / per;
    const int b = bh / a.Hkv, h = bh % a.Hkv, j0 = (blockIdx.x % per) * kWKeys, tid = threadIdx.x;
    const int len = own_length(a, b), j = j0 + tid;
    const int64_t at = ((int64_t)b * a.Hkv + h) * a.T + j;
    if (j0 >= len) {
        if (j < a.T) scores_out[at] = scores[at];
        return;
    }
    const float* kb = static_cast<const float*>(a.k) + b * a.k_b + h * a.k_h;
    for (int i = tid; i < kWKeys * (D / 8); i += kWKeys) {
        const int r = i / (D / 8), c = i % (D / 8);
        float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (j0 + r < len) load8<float>(kb + (int64_t)(j0 + r) * a.k_t + c * 8, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) sk[r * LDK + c * 8 + e] = x[e];
    }
    const int nrows = a.Tq * a.G;
    const float4* k4 = reinterpret_cast<const float4*>(sk + tid * LDK);
    float w = 0.0f;
    for (int r0 = 0; r0 < nrows; r0 += kWRows) {
        __syncthreads();
        for (int i = tid; i < kWRows * (D / 8); i += kWKeys) {
            const int r = r0 + i / (D / 8), c = i % (D / 8);
            float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (r < nrows)
                load8<float>(static_cast<const float*>(a.q) + b * a.q_b + r / a.G * a.q_t + (h * (int64_t)a.G + r % a.G) * a.q_h +
                             c * 8,
                         x);
#pragma unroll
            for (int e = 0; e < 8; ++e) sq[(i / (D / 8)) * D + c * 8 + e] = x[e];
        }
        if (tid < kWRows)
            slse[tid] = r0 + tid < nrows
                            ? a.lse2[row_index(a, (int64_t)b * a.Tq + (r0 + tid) / a.G, h, (r0 + tid) % a.G)]
                            : 0.0f;
        __syncthreads();
        float s[kWRows] = {};
#pragma unroll 4
        for (int c = 0; c < D / 4; ++c) {
            const float4 kk = k4[c];
#pragma unroll
            for (int u = 0; u < kWRows; ++u) {
                const float4 qq = reinterpret_cast<const float4*>(sq + u * D)[c];
                s[u] = fmaf(qq.x, kk.x, fmaf(qq.y, kk.y, fmaf(qq.z, kk.z, fmaf(qq.w, kk.w, s[u]))));
            }
        }
#pragma unroll
        for (int u = 0; u < kWRows; ++u) {
            const int r = r0 + u;
            if (r < nrows && j < len - a.Tq + r / a.G + 1) w += exp2f(s[u] * a.scale_log2 - slse[u]);
        }
    }
    if (j < a.T) scores_out[at] = scores[at] + w;
}

template <int D>
int weights_launch(const PrefixArgs& a, const float* scores, float* scores_out, cudaStream_t stream) {
    const int smem = (kWKeys * (D + 4) + kWRows * D) * 4;
    if (!allow_kernel<own_weights_kernel<D>>(smem)) return LSA_ERR_CUDA;
    const int64_t grid = ((int64_t)a.T + kWKeys - 1) / kWKeys * a.Hkv * a.B;
    if (grid > INT32_MAX) return LSA_ERR_SIZE;
    own_weights_kernel<D><<<(unsigned)grid, kWKeys, smem, stream>>>(a, scores, scores_out);
    LSA_LAUNCH_CHECK();
    return LSA_OK;
}

}  // namespace

int launch_own_weights(const PrefixArgs& a, int D, const float* scores, float* scores_out, cudaStream_t stream) {
    return D == 128 ? weights_launch<128>(a, scores, scores_out, stream)
                    : weights_launch<64>(a, scores, scores_out, stream);
}

}  // namespace lsa
