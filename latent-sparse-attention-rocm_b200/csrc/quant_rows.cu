// quant_rows.cu - attention over the 8-bit paged cache for few rows, and its sparse read (sm_100a).
// quant.cuh has the formulas.
//
// A work item is at most 16 query rows of one KV head (a sequence's last tokens; of the read one token's G query
// heads) x a range of keys. The keys' bytes bound it: 2 D a key and head. So nothing waits for a neighbour in the
// main loop: each of a CTA's four warps copies its own tiles of 32 keys (cp.async, 16 bytes, kRing tiles in
// flight) and runs its own online softmax on them. S = Q K^T and O += P V by mma.sync.m16n8k16 in fp16 (one
// M = 16 tile holds all rows), the codes made halves in registers on their way into the fragments, which
// is exact:
//   K: a lane takes 16 bytes of key g = lane / 4 at a time, four consecutive bytes a k-step; Q's fragments are
//      loaded in the same order of D, which a product does not see.
//   V: a lane takes D / 8 bytes of four keys and makes pairs of two keys' codes (the fragment's order) by byte
//      permutes; a k-step's eight columns are then D / 8 apart, and the output's columns are put back at the end.
// Q is made fp16 as well: bf16 rows by an exact power of two that brings their largest value to [2^8, 2^9)
// (what is 2^-22 of it or less loses bits, 2^-33 of it at most), back in the row's factor.
// P (at most 1) is rounded to fp16 for its product, times 2^15, the most that it holds: 2^-40 of a row's largest
// is kept. Sums, maxima and joins are fp32.
#include <type_traits>

#include "quant.cuh"
#include "umma.cuh"

namespace lsa {
namespace {

constexpr int kWarps = 4;
constexpr int kRows = 16;
constexpr int kKeys = 32;  // keys of a warp's tile: one a lane where they are looked up
constexpr float kLift = 15.0f;

template <int D> struct QuantShape {
    static constexpr int kRing = D == 128 ? 3 : 5;     // tiles in a warp's ring
    static constexpr int kTile = kKeys * D;            // K or V bytes of a tile
    static constexpr int kStage = 2 * kTile + kKeys * 8 + 16;  // + the keys' scales, + which keys are there
    static constexpr int kWarpBytes = (kRing * kStage + 127) / 128 * 128;
    static constexpr int kSmem = kWarps * kWarpBytes + kWarps * kRows * 2 * 4;
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
__device__ __forceinline__ float2 lds_f2(uint32_t addr) {
    float2 r;
    asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(r.x), "=f"(r.y) : "r"(addr) : "memory");
    return r;
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

template <typename T, int CODE, int D, bool LISTS>
__global__ void __launch_bounds__(kWarps * 32, 2) quant_rows_kernel(const QuantArgs a, const int row_tiles) {
    using Sh = QuantShape<D>;
    constexpr int C = D / 16;       // 16-byte chunks of a key
    constexpr int KS = D / 16;      // k-steps of S
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, c = lane & 3;
    grid_wait();
    grid_trigger();
    int item = blockIdx.x;
    const int split = item % a.parts;
    item /= a.parts;
    const int r0 = item % row_tiles * kRows;
    item /= row_tiles;
    const int h = item % a.Hkv, b = item / a.Hkv;
    const int nrows = a.Tq * a.G;
    const int live = nrows - r0 < kRows ? nrows - r0 : kRows;
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
        keys = length - a.Tq + (r0 + live - 1) / a.G + 1;  // that the tile's last row sees
        const int64_t room = (int64_t)a.M << a.shift;
        keys = keys < 0 ? 0 : (keys > room ? (int)room : keys);
    }
    int k0, k1;
    {
        const int64_t units = (keys + kWarps * kKeys - 1) / (kWarps * kKeys);
        const int64_t u0 = units * split / a.parts * (kWarps * kKeys), u1 = units * (split + 1) / a.parts * (kWarps * kKeys);
        k0 = (int)(u0 < keys ? u0 : keys), k1 = (int)(u1 < keys ? u1 : keys);
    }
    const int32_t* table = a.table + trow * a.table_ld;
    const int32_t* list = LISTS ? a.lists + (int64_t)b * a.W : nullptr;
    const uint32_t ring = smem_u32(smem) + warp * Sh::kWarpBytes;
    const int tiles = k1 - k0 > warp * kKeys ? (k1 - k0 - warp * kKeys + kWarps * kKeys - 1) / (kWarps * kKeys) : 0;

    // tile i of this warp: keys k0 + (warp + 4 i) 32 ..; a lane looks its key up, then the warp copies the rows
    auto copy = [&](int i) {
        if (i < tiles) {
            const int key = k0 + (warp + kWarps * i) * kKeys + lane;
            int pos = key;
            bool in = key < k1;
            if (LISTS) {
                pos = in ? list[key] : 0;
                in = in && pos >= 0 && pos < length && (pos >> a.shift) < a.M;
            }
            const int page = in ? table[pos >> a.shift] : -1;
            in = in && page >= 0 && page < a.pages;
            const int64_t head = in ? (int64_t)page * a.Hkv + h : 0;
            // row of the pool (below 2^31: the entry point checks); a key that is not there is not read
            const int row = in ? (int)((head << a.shift) + (pos & ((1 << a.shift) - 1))) : -1;
            const uint32_t stage = ring + (i % Sh::kRing) * Sh::kStage;
            const uint32_t scales = stage + 2 * Sh::kTile;
            cp_async4(scales + lane * 8, a.ks + head, in ? 4u : 0u);
            cp_async4(scales + lane * 8 + 4, a.vs + head, in ? 4u : 0u);
            const uint32_t there = __ballot_sync(0xFFFFFFFFu, in);
            if (lane == 0) asm volatile("st.shared.b32 [%0], %1;" ::"r"(scales + kKeys * 8), "r"(there) : "memory");
#pragma unroll
            for (int rr = 0; rr < kKeys; rr += 32 / C) {
                const int r = rr + lane / C, ch = lane % C;
                const int from = __shfl_sync(0xFFFFFFFFu, row, r);
                const int64_t at = (int64_t)(from < 0 ? 0 : from) * D + ch * 16;
                cp_async16(stage + k_at<D>(r, ch), a.k8 + at, from < 0 ? 0u : 16u);
                cp_async16(stage + Sh::kTile + v_at<D>(r, ch), a.v8 + at, from < 0 ? 0u : 16u);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < Sh::kRing - 1; ++i) copy(i);

    // Q fragments: rows r0 + g and r0 + g + 8; k-step kk's four values of a lane are D's
    // 16 (c + 4 (kk / 4)) + 4 (kk % 4) + 0..3
    uint32_t qf[KS][4];
    int limit[2];
    float factor[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int r = r0 + g + 8 * u;
        const int tok = r / a.G;
        limit[u] = r >= nrows ? 0 : (LISTS ? k1 : length - a.Tq + tok + 1);
        const T* src = static_cast<const T*>(a.q) + b * a.q_b + tok * a.q_t + (h * (int64_t)a.G + r - tok * a.G) * a.q_h;
        uint2 raw[KS];
#pragma unroll
        for (int kk = 0; kk < KS; ++kk)
            raw[kk] = r < nrows ? *reinterpret_cast<const uint2*>(src + 16 * (c + 4 * (kk >> 2)) + 4 * (kk & 3))
                                : make_uint2(0, 0);
        factor[u] = a.scale_log2;
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            uint32_t top = 0;  // largest magnitude's bits, as a bf16
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
                const uint32_t w[2] = {raw[kk].x, raw[kk].y};
#pragma unroll
                for (int e = 0; e < 2; ++e) top = max(top, max(w[e] & 0x7FFFu, (w[e] >> 16) & 0x7FFFu));
            }
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            const int e = (int)(top >> 7);  // biased exponent; zero, and infinities and NaN, stay as they are
            const int up = e == 0 || e == 255 ? 0 : min(8 - (e - 127), 100);
            const float f = __uint_as_float((uint32_t)(up + 127) << 23);
            factor[u] *= __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
                qf[kk][u] = pack_half(__uint_as_float(raw[kk].x << 16) * f, __uint_as_float(raw[kk].x & 0xFFFF0000u) * f);
                qf[kk][u + 2] = pack_half(__uint_as_float(raw[kk].y << 16) * f, __uint_as_float(raw[kk].y & 0xFFFF0000u) * f);
            }
        } else {
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) qf[kk][u] = raw[kk].x, qf[kk][u + 2] = raw[kk].y;
        }
    }
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

    for (int i = 0; i < tiles; ++i) {
        copy(i + Sh::kRing - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(Sh::kRing - 1) : "memory");
        __syncwarp();
        const uint32_t ks = ring + (i % Sh::kRing) * Sh::kStage, vs = ks + Sh::kTile, scales = vs + Sh::kTile;
        const int key0 = k0 + (warp + kWarps * i) * kKeys;
        const uint32_t there = lds32(scales + kKeys * 8);
        float s[4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[t][e] = 0.0f;
#pragma unroll
            for (int hh = 0; hh < KS / 4; ++hh) {
                uint32_t w[4];
                lds_words<4>(w, ks + k_at<D>(t * 8 + g, c + 4 * hh));
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    mma_f16(s[t], qf[4 * hh + kk], halves_of<CODE>(w[kk], 0), halves_of<CODE>(w[kk], 1));
            }
        }
        // logits with the value scale in the exponent; -inf where there is no key, or none for the row
        float inv[4][2], mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int n = t * 8 + 2 * c + e;
                const float2 sc = lds_f2(scales + n * 8);
                const float v = fmaxf(sc.y, 8.6736174e-19f);  // 2^-60
                const float lv = __log2f(v);
                inv[t][e] = __frcp_rn(v);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float& x = s[t][2 * u + e];
                    const bool seen = (there >> n & 1u) && (LISTS || key0 + n < limit[u]);
                    x = seen ? fmaf(x * sc.x, factor[u], lv) : -INFINITY;
                    mx[u] = fmaxf(mx[u], x);
                }
            }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
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
                for (int d = 0; d < D / 8; ++d) o[d][2 * u] *= alpha, o[d][2 * u + 1] *= alpha;
            }
        }
        uint32_t p[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float base = m[u] == -INFINITY ? 0.0f : m[u];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const float p0 = ex2_approx((s[t][2 * u] - base) + kLift), p1 = ex2_approx((s[t][2 * u + 1] - base) + kLift);
                l[u] = fmaf(p0, inv[t][0], fmaf(p1, inv[t][1], l[u]));
                p[t >> 1][u + 2 * (t & 1)] = pack_half(p0, p1);
            }
        }
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            // keys 16 kk + 2c, + 1, + 8, + 9 of the tile
            constexpr int NW = D / 32;  // words of a key a lane takes: D's (D / 8) g ..
            uint32_t w[4][NW];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int r = 16 * kk + 2 * c + (x & 1) + 8 * (x >> 1);
                if constexpr (D == 128)
                    lds_words<NW>(w[x], vs + v_at<D>(r, g));
                else
                    lds_words<NW>(w[x], vs + v_at<D>(r, g >> 1) + (g & 1) * 8);
            }
#pragma unroll
            for (int j = 0; j < NW; ++j) {
                const uint32_t lo0 = __byte_perm(w[0][j], w[1][j], 0x5140), lo1 = __byte_perm(w[0][j], w[1][j], 0x7362);
                const uint32_t hi0 = __byte_perm(w[2][j], w[3][j], 0x5140), hi1 = __byte_perm(w[2][j], w[3][j], 0x7362);
                mma_f16(o[4 * j], p[kk], halves_of<CODE>(lo0, 0), halves_of<CODE>(hi0, 0));
                mma_f16(o[4 * j + 1], p[kk], halves_of<CODE>(lo0, 1), halves_of<CODE>(hi0, 1));
                mma_f16(o[4 * j + 2], p[kk], halves_of<CODE>(lo1, 0), halves_of<CODE>(hi1, 0));
                mma_f16(o[4 * j + 3], p[kk], halves_of<CODE>(lo1, 1), halves_of<CODE>(hi1, 1));
            }
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
        // o[i]'s columns 2c and 2c + 1 are D's (D / 8) 2c + i and (D / 8)(2c + 1) + i
        float* line = so + (g + 8 * u) * D + (D / 8) * 2 * c;
#pragma unroll
        for (int i = 0; i < D / 8; i += 4) {
            *reinterpret_cast<float4*>(line + i) = make_float4(o[i][2 * u], o[i + 1][2 * u], o[i + 2][2 * u], o[i + 3][2 * u]);
            *reinterpret_cast<float4*>(line + D / 8 + i) =
                make_float4(o[i][2 * u + 1], o[i + 1][2 * u + 1], o[i + 2][2 * u + 1], o[i + 3][2 * u + 1]);
        }
        if (c == 0) sml[warp * kRows + g + 8 * u] = make_float2(m[u], l[u]);
    }
    __syncthreads();
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
            const float f = ml.y == 0.0f ? 0.0f : exp2f(ml.x - top);  // NaN passes on
            const float4 y = *reinterpret_cast<const float4*>(smem + w * Sh::kWarpBytes + (r * D + col) * 4);
            total = fmaf(f, ml.y, total);
            x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y), x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w);
        }
        const float norm = total == 0.0f ? 0.0f : 1.0f / total;
        x.x *= norm, x.y *= norm, x.z *= norm, x.w *= norm;
        const float lse = total == 0.0f ? -INFINITY : top + (log2f(total) - kLift);
        const int tok = (r0 + r) / a.G;
        const int64_t rid = ((int64_t)b * a.Tq + tok) * a.Hq + (int64_t)h * a.G + (r0 + r - tok * a.G);
        if (a.parts == 1) {
            T* dst = static_cast<T*>(a.out) + rid * D + col;
            const T y[4] = {from_f32<T>(x.x), from_f32<T>(x.y), from_f32<T>(x.z), from_f32<T>(x.w)};
            *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(y);
            if (col == 0 && a.lse) a.lse[rid] = lse * 0.69314718055994531f;
        } else {
            const int64_t at = (int64_t)split * a.rows + rid;
            *reinterpret_cast<float4*>(a.part_o + at * D + col) = x;
            if (col == 0) a.part_lse[at] = lse;
        }
    }
}

// The parts of a row joined: a CTA a row, a warp every fourth part.
template <typename T, int D>
__global__ void __launch_bounds__(128) quant_join_kernel(const QuantArgs a) {
    constexpr int V = D / 32;
    __shared__ float so[4][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_wait();
    grid_trigger();
    const int64_t rid = blockIdx.x;
    float lse[3], top = -INFINITY;  // at most 96 parts, 32 a load
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const int part = i * 32 + lane;
        lse[i] = part < a.parts ? a.part_lse[part * a.rows + rid] : -INFINITY;
        top = fmaxf(top, lse[i]);
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, off));
    float total = 0.0f, o[V];
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = 0.0f;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        // NaN passes on; a part without a key is not read
        const float f = lse[i] == -INFINITY ? 0.0f : exp2f(lse[i] - (top == -INFINITY ? 0.0f : top));
        float w = f;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) w += __shfl_xor_sync(0xFFFFFFFFu, w, off);
        total += w;
        const int n = a.parts - i * 32 < 32 ? a.parts - i * 32 : 32;
#pragma unroll 4
        for (int j = warp; j < n; j += 4) {
            const float fj = __shfl_sync(0xFFFFFFFFu, f, j);
            if (fj == 0.0f) continue;
            const float* src = a.part_o + ((int64_t)(i * 32 + j) * a.rows + rid) * D + lane * V;
            if constexpr (V == 4) {
                const float4 y = *reinterpret_cast<const float4*>(src);
                o[0] = fmaf(fj, y.x, o[0]), o[1] = fmaf(fj, y.y, o[1]), o[2] = fmaf(fj, y.z, o[2]), o[3] = fmaf(fj, y.w, o[3]);
            } else {
                const float2 y = *reinterpret_cast<const float2*>(src);
                o[0] = fmaf(fj, y.x, o[0]), o[1] = fmaf(fj, y.y, o[1]);
            }
        }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) so[warp][lane * V + e] = o[e];
    __syncthreads();
    const int col = threadIdx.x;
    if (col < D) {
        const float x = (so[0][col] + so[1][col]) + (so[2][col] + so[3][col]);
        static_cast<T*>(a.out)[rid * D + col] = from_f32<T>(total == 0.0f ? 0.0f : x / total);
    }
    if (threadIdx.x == 0 && a.lse)
        a.lse[rid] = total == 0.0f ? -INFINITY : (top + log2f(total)) * 0.69314718055994531f;
}

template <typename T, int CODE, int D, bool LISTS>
int launch(const QuantArgs& a, int row_tiles, unsigned grid, cudaStream_t stream) {
    if (!allow_kernel<quant_rows_kernel<T, CODE, D, LISTS>>(QuantShape<D>::kSmem)) return LSA_ERR_CUDA;
    return launch_after(quant_rows_kernel<T, CODE, D, LISTS>, dim3(grid), kWarps * 32, QuantShape<D>::kSmem, stream, a,
                        row_tiles);
}
template <typename T, int CODE, int D>
int launch(const QuantArgs& a, int row_tiles, unsigned grid, cudaStream_t stream) {
    return a.lists ? launch<T, CODE, D, true>(a, row_tiles, grid, stream)
                   : launch<T, CODE, D, false>(a, row_tiles, grid, stream);
}
template <typename T> int launch(const QuantArgs& a, int code, int D, int row_tiles, unsigned grid, cudaStream_t stream) {
    if (code == kE4M3)
        return D == 128 ? launch<T, kE4M3, 128>(a, row_tiles, grid, stream) : launch<T, kE4M3, 64>(a, row_tiles, grid, stream);
    return D == 128 ? launch<T, kInt8, 128>(a, row_tiles, grid, stream) : launch<T, kInt8, 64>(a, row_tiles, grid, stream);
}

}  // namespace

int launch_quant_rows(const QuantArgs& a, int dtype, int code, int D, cudaStream_t stream) {
    const int row_tiles = (a.Tq * a.G + kRows - 1) / kRows;
    const int64_t items = (int64_t)a.B * a.Hkv * row_tiles * a.parts;
    if (items > INT32_MAX) return LSA_ERR_SIZE;
    return dtype == kBF16 ? launch<__nv_bfloat16>(a, code, D, row_tiles, (unsigned)items, stream)
                          : launch<__half>(a, code, D, row_tiles, (unsigned)items, stream);
}

int launch_quant_join(const QuantArgs& a, int dtype, int D, cudaStream_t stream) {
    if (a.rows > INT32_MAX) return LSA_ERR_SIZE;
    const dim3 grid((unsigned)a.rows);
    if (dtype == kBF16)
        return D == 128 ? launch_after(quant_join_kernel<__nv_bfloat16, 128>, grid, 128, 0, stream, a)
                        : launch_after(quant_join_kernel<__nv_bfloat16, 64>, grid, 128, 0, stream, a);
    return D == 128 ? launch_after(quant_join_kernel<__half, 128>, grid, 128, 0, stream, a)
                    : launch_after(quant_join_kernel<__half, 64>, grid, 128, 0, stream, a);
}

}  // namespace lsa
