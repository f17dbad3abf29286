// prefix_rows.cu - the shared-prefix attention of few rows: decode steps (sm_100a).
//
// A work item is at most 16 query rows of one KV head (a sequence's decode rows against its own
// cache, or a small batch's against the prefix) x a range of keys; a sequence with up to 64 rows and
// a short cache is several items that read the same keys, from L2 after the first. The keys' bytes bound it: 512
// bytes of K and V per key and head (D = 128, 16 bits) against 16 rows of arithmetic. So nothing
// waits for a neighbour in the main loop: each of a CTA's four warps copies its own tiles of 16
// keys (cp.async, 16 bytes, three stages of 8 KB in flight per warp, two CTAs an SM) and runs its
// own online softmax on them: S = Q K^T and O += P V by mma.sync.m16n8k16 (one M = 16 tile holds
// all rows; a 128-row tcgen05 tile would be 1/8 full or less and pass through TMEM), maximum and
// sum in fp32 registers, P rounded to the inputs' type for its product (fp16: times 2^15 first, the most
// that it holds, or a weight below 2^-25 of the maximum would leave O and stay in the sum; the factor is in
// both and cancels). The warps join through
// shared memory at the end. Measured (32 / 8 heads, D 128, bf16, called in a loop, the join of the parts
// included): 48 ragged caches of up to 8191 keys, 1.2 GB, 188 us = 6.4 TB/s, 97 % of the measured copy rate; 16 of
// 6144 keys 79 us = 5.1 TB/s; one of 24576 keys 23 us, of which 15 are the memory's. Keys at or past the range's
// end are zero-filled by the copy, so what an unwritten slot holds is never used.
#include "prefix.cuh"
#include "umma.cuh"

namespace lsa {
namespace {

constexpr int kWarps = 4;
constexpr int kRows = 16;
constexpr int kKeys = 16;  // keys of a warp's tile
constexpr int kRing = 3;   // tiles in a warp's ring

template <typename T> constexpr float kLift = 0.0f;  // log2 of the factor that the weights carry
template <> constexpr float kLift<__half> = 15.0f;

template <int D> struct RowsShape {
    static constexpr int kTile = kKeys * D * 2;          // K or V bytes of a tile
    static constexpr int kWarpBytes = kRing * 2 * kTile; // at least the 16 x D fp32 of the join
    static constexpr int kSmem = kWarps * kWarpBytes + kWarps * kRows * 2 * 4;
    static_assert(kWarpBytes >= kRows * D * 4, "the join reuses a warp's ring");
};

// 16-byte copy under an L2 policy; src_bytes 0 zero-fills without reading.
__device__ __forceinline__ void cp_async16_hint(uint32_t dst, const void* src, uint32_t src_bytes, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src),
                 "r"(src_bytes), "l"(policy)
                 : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                      __nv_bfloat16*) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half*) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pk16(float a, float b, __nv_bfloat16*) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pk16(float a, float b, __half*) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}

template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32, 2) prefix_rows_kernel(const PrefixArgs a, const RowsPlan rp) {
    using Sh = RowsShape<D>;
    constexpr int C = D / 8;  // 16-byte chunks of a row
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // Behind the call's tensor-core kernel (which waited for everything before the call) this one
    // starts on what that one leaves free; what follows needs both, so one CTA, the last, waits for it
    // at its end (a wait of every CTA would keep their places until then).
    if (!rp.follows) grid_wait();
    grid_trigger();
    int item = blockIdx.x;
    const bool own = item >= rp.prefix_items;
    int b = 0, h, part, nrows, r0 = 0, k0, k1, len = 0;
    if (!own) {
        const int split = item % a.Sp;
        h = item / a.Sp;
        part = split;
        nrows = a.B * a.Tq * a.G;
        split_range(a.P, split, a.Sp, kWarps * kKeys, &k0, &k1);
    } else {
        item -= rp.prefix_items;
        const int split = item % a.So;
        item /= a.So;
        r0 = item % rp.own_tiles * kRows;
        item /= rp.own_tiles;
        h = item % a.Hkv, b = item / a.Hkv;
        part = a.parts_p + split;
        nrows = a.Tq * a.G;
        len = own_length(a, b);
        split_range(len, split, a.So, kWarps * kKeys, &k0, &k1);
    }
    const T* kb = static_cast<const T*>(own ? a.k : a.kp) + (own ? b * a.k_b + h * a.k_h : h * a.kp_h);
    const T* vb = static_cast<const T*>(own ? a.v : a.vp) + (own ? b * a.v_b + h * a.v_h : h * a.vp_h);
    const int64_t kt = own ? a.k_t : a.kp_t, vt = own ? a.v_t : a.vp_t;
    const uint32_t ring = smem_u32(smem) + warp * Sh::kWarpBytes;

    // tile i of this warp: keys k0 + (warp + 4 i) 16 ..; a lane copies chunk `lane % C` of every
    // (32 / C)-th row
    const int tiles = k1 - k0 > warp * kKeys ? (k1 - k0 - warp * kKeys + kWarps * kKeys - 1) / (kWarps * kKeys) : 0;
    const int lc = lane % C, lr = lane / C;
    // keys that nothing reads again leave L2 before the logits do
    uint64_t policy;
    if (own && rp.logits && rp.own_tiles == 1)
        asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    else
        asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
    auto copy = [&](int i) {
        if (i < tiles) {
            const int key0 = k0 + (warp + kWarps * i) * kKeys;
            const uint32_t dst = ring + (i % kRing) * 2 * Sh::kTile;
#pragma unroll
            for (int rr = 0; rr < kKeys; rr += 32 / C) {
                const int row = rr + lr, key = key0 + row;
                const bool in = key < k1;
                const int64_t at = in ? key : k0;
                const uint32_t to = dst + row * D * 2 + ((lc ^ (row & 7)) << 4);
                cp_async16_hint(to, kb + at * kt + lc * 8, in ? 16u : 0u, policy);
                cp_async16_hint(to + Sh::kTile, vb + at * vt + lc * 8, in ? 16u : 0u, policy);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) copy(i);

    // Q fragments: rows r0 + lane / 4 and r0 + lane / 4 + 8
    uint32_t qf[D / 16][4];
    int limit[2];
    const int quad = lane >> 2, qc = (lane & 3) * 2;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int r = r0 + quad + 8 * u;
        const int tok = r / a.G;
        limit[u] = r >= nrows ? 0 : (own ? len - a.Tq + tok + 1 : k1);
        const int64_t bt = (int64_t)b * a.Tq + tok;
        const T* src = static_cast<const T*>(a.q) + bt / a.Tq * a.q_b + bt % a.Tq * a.q_t +
                       (h * (int64_t)a.G + r - tok * a.G) * a.q_h;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            qf[kk][u] = r < nrows ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + qc) : 0u;
            qf[kk][u + 2] = r < nrows ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + 8 + qc) : 0u;
        }
    }
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float* logits = own && rp.logits
                        ? rp.logits + (((int64_t)b * a.Hkv + h) * nrows + r0 + quad) * rp.pitch
                        : nullptr;

    for (int i = 0; i < tiles; ++i) {
        copy(i + kRing - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 1) : "memory");
        __syncwarp();
        const uint32_t ks = ring + (i % kRing) * 2 * Sh::kTile, vs = ks + Sh::kTile;
        float s[2][4] = {};
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t kf[4];
            const int row = (lane & 7) + ((lane >> 4) << 3), c = 2 * kk + ((lane >> 3) & 1);
            ldsm4(kf, ks + row * D * 2 + ((c ^ (row & 7)) << 4));
            mma16(s[0], qf[kk], kf[0], kf[1], (T*)nullptr);
            mma16(s[1], qf[kk], kf[2], kf[3], (T*)nullptr);
        }
        const int key0 = k0 + (warp + kWarps * i) * kKeys;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = key0 + t * 8 + qc + (e & 1);
                s[t][e] = key < k1 && key < limit[e >> 1] ? s[t][e] * a.scale_log2 : -INFINITY;
            }
        if (logits) {  // whole 32-byte sectors: four lanes a row; the rows' pitch covers a last, ragged tile
#pragma unroll
            for (int u = 0; u < 2; ++u)
                if (r0 + quad + 8 * u < nrows)
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        *reinterpret_cast<float2*>(logits + (int64_t)8 * u * rp.pitch + key0 + t * 8 + qc) =
                            make_float2(s[t][2 * u], s[t][2 * u + 1]);
        }
        float mx[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            mx[u] = fmaxf(fmaxf(s[0][2 * u], s[0][2 * u + 1]), fmaxf(s[1][2 * u], s[1][2 * u + 1]));
            mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xFFFFFFFFu, mx[u], 1));
            mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xFFFFFFFFu, mx[u], 2));
        }
        if (__any_sync(0xFFFFFFFFu, mx[0] > m[0] || mx[1] > m[1])) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float mn = fmaxf(m[u], mx[u]);
                const float alpha = mn == -INFINITY ? 0.0f : ex2_approx(m[u] - mn);
                m[u] = mn;
                l[u] *= alpha;
#pragma unroll
                for (int d = 0; d < D / 8; ++d) {
                    o[d][2 * u] *= alpha;
                    o[d][2 * u + 1] *= alpha;
                }
            }
        }
        uint32_t p[4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float base = m[u] == -INFINITY ? 0.0f : m[u];
            auto weight = [&](float x) {  // at most 2^kLift, exactly
                return ex2_approx(kLift<T> == 0.0f ? x - base : (x - base) + kLift<T>);
            };
            const float p0 = weight(s[0][2 * u]), p1 = weight(s[0][2 * u + 1]);
            const float p2 = weight(s[1][2 * u]), p3 = weight(s[1][2 * u + 1]);
            l[u] += (p0 + p1) + (p2 + p3);
            p[u] = pk16(p0, p1, (T*)nullptr);
            p[u + 2] = pk16(p2, p3, (T*)nullptr);
        }
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            uint32_t vf[4];
            const int row = (lane & 7) + (((lane >> 3) & 1) << 3), c = 2 * d + (lane >> 4);
            ldsm4_t(vf, vs + row * D * 2 + ((c ^ (row & 7)) << 4));
            mma16(o[2 * d], p, vf[0], vf[1], (T*)nullptr);
            mma16(o[2 * d + 1], p, vf[2], vf[3], (T*)nullptr);
        }
        __syncwarp();  // the tile's slot is refilled next
    }
    cp_async_wait_all();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        l[u] += __shfl_xor_sync(0xFFFFFFFFu, l[u], 1);
        l[u] += __shfl_xor_sync(0xFFFFFFFFu, l[u], 2);
    }
    // join the warps: each leaves its sums in its own ring, (m, l) after the rings
    __syncwarp();
    float* so = reinterpret_cast<float*>(smem + warp * Sh::kWarpBytes);
    float2* sml = reinterpret_cast<float2*>(smem + kWarps * Sh::kWarpBytes);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int d = 0; d < D / 8; ++d)
            *reinterpret_cast<float2*>(so + (quad + 8 * u) * D + d * 8 + qc) = make_float2(o[d][2 * u], o[d][2 * u + 1]);
        if ((lane & 3) == 0) sml[warp * kRows + quad + 8 * u] = make_float2(m[u], l[u]);
    }
    __syncthreads();
    const int live = nrows - r0 < kRows ? nrows - r0 : kRows;
    for (int i = threadIdx.x; i < live * (D / 4); i += kWarps * 32) {
        const int r = i / (D / 4), c = i % (D / 4) * 4;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sml[w * kRows + r].x);
        float total = 0.0f;
        float4 x = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float2 ml = sml[w * kRows + r];
            const float f = ml.y == 0.0f ? 0.0f : exp2f(ml.x - top);  // NaN passes on
            const float4 y = *reinterpret_cast<const float4*>(smem + w * Sh::kWarpBytes + (r * D + c) * 4);
            total = fmaf(f, ml.y, total);
            x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y), x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w);
        }
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        const int tok = (r0 + r) / a.G;
        const int64_t rid = row_index(a, (int64_t)b * a.Tq + tok, h, r0 + r - tok * a.G);
        const int64_t at = (int64_t)part * a.rows + rid;
        if (c == 0) a.part_lse[at] = total == 0.0f ? -INFINITY : top + (log2f(total) - kLift<T>);
        *reinterpret_cast<float4*>(a.part_o + at * D + c) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
    }
    if (rp.follows && blockIdx.x == gridDim.x - 1) grid_wait();
}

template <typename T, int D>
int launch(const PrefixArgs& a, const RowsPlan& rp, unsigned grid, cudaStream_t stream) {
    if (!allow_kernel<prefix_rows_kernel<T, D>>(RowsShape<D>::kSmem)) return LSA_ERR_CUDA;
    return launch_after(prefix_rows_kernel<T, D>, dim3(grid), kWarps * 32, RowsShape<D>::kSmem, stream, a, rp);
}

}  // namespace

int launch_prefix_rows(const PrefixArgs& a, const RowsPlan& rp, int dtype, int D, cudaStream_t stream) {
    const int64_t items = (int64_t)rp.prefix_items + rp.own_items;
    if (items == 0) return LSA_OK;
    if (items > INT32_MAX) return LSA_ERR_SIZE;
    const unsigned grid = (unsigned)items;
    if (dtype == kBF16)
        return D == 128 ? launch<__nv_bfloat16, 128>(a, rp, grid, stream)
                        : launch<__nv_bfloat16, 64>(a, rp, grid, stream);
    return D == 128 ? launch<__half, 128>(a, rp, grid, stream) : launch<__half, 64>(a, rp, grid, stream);
}

}  // namespace lsa
