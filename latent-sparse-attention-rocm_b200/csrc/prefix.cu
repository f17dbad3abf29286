// prefix.cu - attention over a shared prefix and each sequence's own cache: the entry points,
// the fp32 kernel and the join of the parts (sm_100a). prefix.cuh has the formulas.
//
// Which kernel reads which segment (make_plan): fp32 inputs the FMA-pipe kernel here; 16-bit inputs
// segments of up to 16 rows a KV head (64 where the keys are few) the few-row kernel, others the
// tensor-core kernel; sequences whose rows fill tiles by themselves read prefix and own keys in one
// item and, but for the last round of tiles, write the output at once.
#include <math.h>

#include "prefix.cuh"

namespace lsa {
namespace {

constexpr int kSMs = 148;
constexpr int kSimtRows = 16;  // rows of a work item
constexpr int kSimtKeys = 32;  // keys of a tile: one per lane
constexpr int kSimtWarps = 8;
constexpr int kFewRows = 16;   // rows of a KV head in an item of the few-row kernel
constexpr int kMostFew = 64;   // rows of a sequence and KV head that it takes at most

template <int D>
__device__ __forceinline__ void stage_rows(float* dst, int ld, const float* src, int64_t stride, int rows, int live) {
    for (int i = threadIdx.x; i < rows * (D / 8); i += blockDim.x) {
        const int r = i / (D / 8), c = i % (D / 8);
        float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (r < live) load8<float>(src + r * stride + c * 8, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) dst[r * ld + c * 8 + e] = x[e];
    }
}

// fp32 inputs. One work item: up to 16 rows of a KV head x a range of keys, on the FMA pipes. A
// warp holds two rows; a lane scores one key of a 32-key tile for both, the warp's running
// maximum and sum follow the tile, and a lane then owns D / 32 output columns. Rows past a
// sequence's length are staged as zeros, so what an unwritten slot holds is never used. What bounds it: a
// tile's loads are waited for at a barrier with nothing in flight beside them, and 16 rows are computed
// whatever is live. Measured (32 / 8 heads, D 128): 16 sequences on 8192 prefix and up to 2048 own keys 286 us, where
// the keys' bytes take 41; 8 x 64 tokens on 4096 keys 2.4 ms.
template <int D>
__global__ void __launch_bounds__(kSimtWarps * 32) prefix_simt_kernel(const PrefixArgs a, int prefix_items, int ptiles,
                                                                      int otiles) {
    constexpr int LDK = D + 4, E = D / 32;
    __shared__ float sq[kSimtRows * D], sk[kSimtKeys * LDK], sv[kSimtKeys * D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int item = blockIdx.x;
    const bool own = item >= prefix_items;
    int b = 0, h, tile, split, part, nrows, k0, k1, len = 0;
    if (!own) {
        split = item % a.Sp, item /= a.Sp;
        tile = item % ptiles, h = item / ptiles;
        part = split;
        nrows = a.B * a.Tq * a.G;
        split_range(a.P, split, a.Sp, kSimtKeys, &k0, &k1);
    } else {
        item -= prefix_items;
        split = item % a.So, item /= a.So;
        tile = item % otiles, item /= otiles;
        h = item % a.Hkv, b = item / a.Hkv;
        part = a.parts_p + split;
        nrows = a.Tq * a.G;
        len = own_length(a, b);
        split_range(len, split, a.So, kSimtKeys, &k0, &k1);
    }
    const int r0 = tile * kSimtRows;
    // q rows (segment order: token, head of the group)
    for (int i = threadIdx.x; i < kSimtRows * (D / 8); i += blockDim.x) {
        const int r = r0 + i / (D / 8), c = i % (D / 8);
        float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (r < nrows) {
            const int64_t tok = (int64_t)b * a.Tq + r / a.G;
            load8<float>(static_cast<const float*>(a.q) + tok / a.Tq * a.q_b + tok % a.Tq * a.q_t +
                         (h * (int64_t)a.G + r % a.G) * a.q_h + c * 8,
                     x);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sq[(i / (D / 8)) * D + c * 8 + e] = x[e];
    }
    const float* kb = static_cast<const float*>(own ? a.k : a.kp) + (own ? b * a.k_b + h * a.k_h : h * a.kp_h);
    const float* vb = static_cast<const float*>(own ? a.v : a.vp) + (own ? b * a.v_b + h * a.v_h : h * a.vp_h);
    const int64_t kt = own ? a.k_t : a.kp_t, vt = own ? a.v_t : a.vp_t;
    // the two rows of this warp: the first key that each does not see
    int limit[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int r = r0 + warp + kSimtWarps * u;
        limit[u] = r >= nrows ? 0 : (own ? len - a.Tq + r / a.G + 1 : k1);
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0, 0}, acc[2][E] = {};
    for (int t0 = k0; t0 < k1; t0 += kSimtKeys) {
        __syncthreads();
        const int live = k1 - t0 < kSimtKeys ? k1 - t0 : kSimtKeys;
        stage_rows<D>(sk, LDK, kb + (int64_t)t0 * kt, kt, kSimtKeys, live);
        stage_rows<D>(sv, D, vb + (int64_t)t0 * vt, vt, kSimtKeys, live);
        __syncthreads();
        float s[2] = {0, 0};
        const float4* k4 = reinterpret_cast<const float4*>(sk + lane * LDK);
#pragma unroll 8
        for (int c = 0; c < D / 4; ++c) {
            const float4 kk = k4[c];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float4 qq = reinterpret_cast<const float4*>(sq + (warp + kSimtWarps * u) * D)[c];
                s[u] = fmaf(qq.x, kk.x, fmaf(qq.y, kk.y, fmaf(qq.z, kk.z, fmaf(qq.w, kk.w, s[u]))));
            }
        }
        float p[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const bool see = lane < live && t0 + lane < limit[u];
            const float x = see ? s[u] * a.scale_log2 : -INFINITY;
            float mx = x;
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, off));
            const float mn = fmaxf(m[u], mx);
            const float base = mn == -INFINITY ? 0.0f : mn;
            const float alpha = exp2f(m[u] - base);
            p[u] = exp2f(x - base);
            float sum = p[u];
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
            l[u] = l[u] * alpha + sum;
            m[u] = mn;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[u][e] *= alpha;
        }
        for (int j = 0; j < live; ++j) {
            const float p0 = __shfl_sync(0xFFFFFFFFu, p[0], j), p1 = __shfl_sync(0xFFFFFFFFu, p[1], j);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float vv = sv[j * D + lane * E + e];
                acc[0][e] = fmaf(p0, vv, acc[0][e]);
                acc[1][e] = fmaf(p1, vv, acc[1][e]);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int r = r0 + warp + kSimtWarps * u;
        if (r >= nrows) continue;
        const int64_t rid = row_index(a, (int64_t)b * a.Tq + r / a.G, h, r % a.G);
        const int64_t at = (int64_t)part * a.rows + rid;
        if (lane == 0) a.part_lse[at] = l[u] == 0.0f ? -INFINITY : m[u] + log2f(l[u]);
        const float inv = l[u] == 0.0f ? 0.0f : 1.0f / l[u];
#pragma unroll
        for (int e = 0; e < E; ++e) a.part_o[at * D + lane * E + e] = acc[u][e] * inv;
    }
}

constexpr int kPer = kMaxParts / 32;  // parts of a row that a lane holds

// The lse of a row from its parts, by one warp (log2 domain; every lane has it).
template <typename F> __device__ __forceinline__ float joined_lse(int parts, F part) {
    const int lane = threadIdx.x & 31;
    float x[kPer], top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        x[i] = -INFINITY;
        if (32 * i < parts && lane + 32 * i < parts) x[i] = part(lane + 32 * i);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        top = fmaxf(top, x[i]);
        sum += x[i] != x[i] ? x[i] : 0.0f;  // a NaN part makes the row NaN
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, off));
    if (top == -INFINITY) top = 0.0f;  // no part has a key: the sum is 0, its logarithm -inf
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (32 * i < parts) sum += exp2f(x[i] - top);
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
    return top + log2f(sum);
}

// Groups of threads that share a weights block's rows: a block of 256 threads takes 1024 / groups keys,
// four a thread. Few rows: one group, the longest runs of keys; more: four, or a thread would
// load them one group of four after another (64 rows: 26 us of latency).
__host__ __device__ __forceinline__ int weight_groups(int nrows) { return nrows > 8 ? 4 : 1; }

constexpr int kHeldLse = 2048;  // parts' lse that a weights block holds in shared memory

// Own keys' weights from the logits that the few-row kernel kept (4 bytes a row and key, 16 for a
// decode step of 4 heads, against the 256 bytes of K that scoring the key again would read):
//   w_j = sum over the rows r that see j of 2^(s_rj - lse_r).
// A key's sum has one order and one writer. The block joins its rows' lse
// itself, beside the blocks that join the output: one launch for both.
__device__ __forceinline__ void own_weights(const PrefixArgs& a, const RowsPlan& rp, int parts,
                                            const float* __restrict__ scores, float* __restrict__ scores_out) {
    __shared__ float slse[kMostFew];
    __shared__ __align__(16) float held[kHeldLse];
    const int nrows = a.Tq * a.G, warp = threadIdx.x >> 5, groups = weight_groups(nrows), quads = 256 / groups;
    const int keys = 4 * quads, per = (int)(((int64_t)a.T + keys - 1) / keys);
    const int64_t bh = blockIdx.x / per;
    const int b = (int)(bh / a.Hkv), h = (int)(bh % a.Hkv);
    const int group = threadIdx.x / quads, quad = threadIdx.x % quads;
    const int len = own_length(a, b), j0 = (blockIdx.x % per) * keys, j = j0 + 4 * quad;
    float old[4] = {0, 0, 0, 0}, w[4] = {0, 0, 0, 0};
    if (group == 0) {
#pragma unroll
        for (int u = 0; u < 4; ++u) old[u] = j + u < a.T ? scores[bh * a.T + j + u] : 0.0f;
    }
    if (j0 < len) {
        // the first rows' logits are on their way while the lse are joined
        const float* src = rp.logits + bh * nrows * rp.pitch + (j < len ? j : j0);
        float4 s[4];
        auto load = [&](int r0) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int r = r0 + u * groups;
                s[u] = __ldcs(reinterpret_cast<const float4*>(src + (r < nrows ? r : 0) * rp.pitch));
            }
        };
        load(group);
        // a warp a row; more than eight rows' parts are fetched together first, not a row at a time
        const bool many = nrows > 8;
        if (many) {
            for (int i = threadIdx.x; i < nrows * parts && i < kHeldLse; i += 256) {
                const int c = i / nrows, r = i - c * nrows, tok = r / a.G;
                held[i] = a.part_lse[c * a.rows + row_index(a, (int64_t)b * a.Tq + tok, h, r - tok * a.G)];
            }
            __syncthreads();
        }
        for (int r = warp; r < nrows; r += 8) {
            const int tok = r / a.G;
            const int64_t row = row_index(a, (int64_t)b * a.Tq + tok, h, r - tok * a.G);
            const float x = joined_lse(parts, [&](int c) {
                const int i = c * nrows + r;
                return many && i < kHeldLse ? held[i] : a.part_lse[c * a.rows + row];
            });
            if ((threadIdx.x & 31) == 0) slse[r] = x;
        }
        __syncthreads();
        for (int r0 = group; r0 < nrows; r0 += 4 * groups) {
            if (r0 != group) load(r0);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (r0 + u * groups >= nrows) break;
                const float l = slse[r0 + u * groups];  // -inf: a row that sees no key, and whose logits are -inf
                w[0] += s[u].x == -INFINITY ? 0.0f : exp2f(s[u].x - l);
                w[1] += s[u].y == -INFINITY ? 0.0f : exp2f(s[u].y - l);
                w[2] += s[u].z == -INFINITY ? 0.0f : exp2f(s[u].z - l);
                w[3] += s[u].w == -INFINITY ? 0.0f : exp2f(s[u].w - l);
            }
        }
        if (groups > 1) {  // the groups' sums in their order
            float4* sums = reinterpret_cast<float4*>(held);
            __syncthreads();
            sums[threadIdx.x] = make_float4(w[0], w[1], w[2], w[3]);
            __syncthreads();
            if (group == 0)
                for (int g = 1; g < groups; ++g) {
                    const float4 x = sums[g * quads + quad];
                    w[0] += x.x, w[1] += x.y, w[2] += x.z, w[3] += x.w;
                }
        }
    }
    if (group != 0) return;
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (j + u < a.T) scores_out[bh * a.T + j + u] = j + u < len ? old[u] + w[u] : old[u];
}

// The parts of a row joined by `spread` warps (1 to 8: more where the rows are few, so that the loads
// of many parts fly together): every lane holds D / 32 columns of a warp's share. The lse of
// all parts are loaded at once, then the parts' columns eight loads at a time; a part without
// a key (lse -inf) has weight zero and its columns, never written, are not read (the heaviest part's
// are, in their place: finite, times zero). The warps' sums add in their order.
template <typename T, int D>
__global__ void __launch_bounds__(256, 4) prefix_finish_kernel(const PrefixArgs a, const TilePlan tp, int parts,
                                                            const RowsPlan rp, unsigned weight_blocks, int spread,
                                                            const float* __restrict__ scores,
                                                            float* __restrict__ scores_out) {
    constexpr int E = D / 32;
    __shared__ float weight[8][kMaxParts], sums[8][D], totals[8];
    grid_trigger();
    grid_wait();
    if (blockIdx.x < weight_blocks) {
        own_weights(a, rp, parts, scores, scores_out);
        return;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % spread;
    int64_t row = (int64_t)(blockIdx.x - weight_blocks) * (8 / spread) + warp / spread;
    const int64_t prow = row;
    if (tp.whole) {  // the rows of the split seq tiles, 256 a tile
        int b, h, tile;
        seq_tile(a, tp, tp.whole + (int)(row >> 8), &b, &h, &tile);
        int tok, g;
        const bool in = tile_row(a, tp, (int)(row >> 7) & 1, (int)(row & 127), &tok, &g);
        tok += tile * 2 * tp.tokens;
        row = in && tok < a.Tq ? row_index(a, (int64_t)b * a.Tq + tok, h, g) : a.rows;
    }
    float acc[E] = {}, total = 0.0f, top = -INFINITY;
    if (row < a.rows) {
        float x[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            x[i] = -INFINITY;
            if (32 * i < parts && lane + 32 * i < parts) x[i] = a.part_lse[(int64_t)(lane + 32 * i) * a.part_rows + prow];
        }
        bool bad = false;
#pragma unroll
        for (int i = 0; i < kPer; ++i) top = fmaxf(top, x[i]), bad = bad || x[i] != x[i];
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, off));
        int best = 0;
#pragma unroll
        for (int i = kPer - 1; i >= 0; --i) {
            if (32 * i >= parts) continue;
            const uint32_t at = __ballot_sync(0xFFFFFFFFu, x[i] == top);
            if (at) best = 32 * i + __ffs(at) - 1;
            weight[warp][32 * i + lane] = top == -INFINITY ? 0.0f : exp2f(x[i] - top);  // past the parts: 0
        }
        __syncwarp();
        if (__any_sync(0xFFFFFFFFu, bad)) {  // a part is NaN: so is the row
            total = NAN;
        } else {
            for (int c0 = 8 * sub; c0 < parts; c0 += 8 * spread) {
                float v[8][E], f[8], some = 0.0f;
#pragma unroll
                for (int u = 0; u < 8; ++u) some += f[u] = weight[warp][c0 + u];
                if (some == 0.0f) continue;
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int c = f[u] > 0.0f ? c0 + u : best;
                    const float* src = a.part_o + ((int64_t)c * a.part_rows + prow) * D + lane * E;
                    if constexpr (E == 4) {
                        const float4 y = __ldcs(reinterpret_cast<const float4*>(src));
                        v[u][0] = y.x, v[u][1] = y.y, v[u][2] = y.z, v[u][3] = y.w;
                    } else {
                        const float2 y = __ldcs(reinterpret_cast<const float2*>(src));
                        v[u][0] = y.x, v[u][1] = y.y;
                    }
                }
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    total += f[u];
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[e] = fmaf(f[u], v[u][e], acc[e]);
                }
            }
        }
    }
    if (spread > 1) {
#pragma unroll
        for (int e = 0; e < E; ++e) sums[warp][lane * E + e] = acc[e];
        if (lane == 0) totals[warp] = total;
        __syncthreads();
        if (sub != 0) return;
        for (int w = warp + 1; w < warp + spread; ++w) {
            total += totals[w];
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += sums[w][lane * E + e];
        }
    }
    if (row >= a.rows) return;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    T* dst = static_cast<T*>(a.out) + row * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) dst[e] = from_f32<T>(acc[e] * inv);
    if (lane == 0) {
        const float y = total == 0.0f ? -INFINITY : top + log2f(total);
        a.lse2[row] = y;
        if (a.lse) a.lse[row] = y * 0.69314718055994531f;
    }
}

}  // namespace

int launch_prefix_simt(const PrefixArgs& a, int D, cudaStream_t stream) {
    const int64_t ptiles = ((int64_t)a.B * a.Tq * a.G + kSimtRows - 1) / kSimtRows;
    const int64_t otiles = ((int64_t)a.Tq * a.G + kSimtRows - 1) / kSimtRows;
    const int64_t pi = a.Sp * ptiles * a.Hkv, oi = (int64_t)a.So * otiles * a.Hkv * a.B;
    if (pi + oi == 0) return LSA_OK;
    if (pi + oi > INT32_MAX) return LSA_ERR_SIZE;
    if (D == 128)
        prefix_simt_kernel<128><<<(unsigned)(pi + oi), kSimtWarps * 32, 0, stream>>>(a, (int)pi, (int)ptiles,
                                                                                        (int)otiles);
    else
        prefix_simt_kernel<64><<<(unsigned)(pi + oi), kSimtWarps * 32, 0, stream>>>(a, (int)pi, (int)ptiles,
                                                                                       (int)otiles);
    LSA_LAUNCH_CHECK();
    return LSA_OK;
}

namespace {

template <typename T>
int finish_d(const PrefixArgs& a, const TilePlan& tp, int D, const RowsPlan& rp, const float* scores,
             float* scores_out, cudaStream_t stream) {
    const int64_t rows = tp.whole ? ((int64_t)a.B * a.Hkv * tp.seq_tiles - tp.whole) * 256 : a.rows;
    const int parts = a.parts_p + a.parts_o;
    int spread = 1;  // warps of a row: no more than the groups of eight parts, while the rows leave SMs idle
    while (spread < 8 && 8 * spread < parts && rows * spread < 16 * kSMs) spread *= 2;
    const int64_t blocks = (rows * spread + 7) / 8;
    const int64_t keys = 1024 / weight_groups(a.Tq * a.G);
    const int64_t weights = rp.logits ? (int64_t)a.B * a.Hkv * (((int64_t)a.T + keys - 1) / keys) : 0;
    if (blocks + weights > INT32_MAX) return LSA_ERR_SIZE;
    auto kern = D == 128 ? prefix_finish_kernel<T, 128> : prefix_finish_kernel<T, 64>;
    return launch_after(kern, dim3((unsigned)(blocks + weights)), 256, 0, stream, a, tp, parts, rp,
                        (unsigned)weights, spread, scores, scores_out);
}

struct Plan {
    int Sp, So, parts_p, parts_o;
    bool simt, logits;  // fp32 inputs; the own keys' logits are kept for their weights
    bool merge;         // some row has parts to join
    TilePlan tile;
    RowsPlan rows;
    int64_t part_rows;  // PrefixArgs::part_rows
};

constexpr int kItemsAPlace = 2;

// Splits of `items` row tiles at most. Parts cost scratch, 132 KB a tile at D 128: split tiles fill no more than
// eight rounds of the SMs (157 MB). With more rounds than that a last, short one is a ninth of the time at most.
constexpr int kMostRounds = 8;
int most_splits(int64_t items) {
    const int64_t s = items ? kMostRounds * kSMs / items : 0;
    return (int)(s < 1 ? 1 : (s < kMaxSplits ? s : kMaxSplits));
}

// Splits of the few-row kernel for `items` of `chunks` steps of 64 keys. One length: 256 CTAs draw the
// memory's whole bandwidth, and more parts cost more to join (one sequence of 24k keys, 8 KV heads: 24.2
// us in 32 parts, 25.6 in 37). Many sequences, of lengths that the host does not know: several
// items a place, so that the long ones even out (one of 64k keys among four of 14k on average: 125 us with
// one item a place, 85 with two).
int few_splits(int64_t items, int64_t chunks, bool ragged) {
    if (chunks == 0) return 0;
    int64_t s = ragged ? (kItemsAPlace * 2 * kSMs + items / 2) / items : 256 / items;
    const int64_t most = items * kMaxSplits >= 256 ? kMaxSplits : 3 * kMaxSplits;
    if (s > most) s = most;
    if (s > chunks / 4) s = chunks / 4;
    return (int)(s < 1 ? 1 : s);
}

Plan make_plan(int dtype, int64_t B, int64_t Tq, int64_t Hkv, int64_t G, int64_t D, int64_t P, int64_t T, bool scored) {
    Plan p = {};
    p.merge = true;
    p.part_rows = B * Tq * Hkv * G;
    p.simt = dtype == kF32;
    if (p.simt) {
        // splits enough that the work items of each segment fill the GPU about four times
        auto splits = [](int64_t items, int64_t keys) -> int {
            if (keys == 0) return 0;
            int64_t s = (4 * kSMs + items - 1) / items;
            const int64_t most = (keys + 255) / 256;
            s = s < most ? s : most;
            return (int)(s < kMaxSplits ? s : kMaxSplits);
        };
        p.parts_p = p.Sp = splits(Hkv * ((B * Tq * G + kSimtRows - 1) / kSimtRows), P);
        p.parts_o = p.So = splits(B * Hkv * ((Tq * G + kSimtRows - 1) / kSimtRows), T);
        return p;
    }
    TilePlan& t = p.tile;
    const int64_t rows = Tq * G;
    const int64_t pc = (P + 127) / 128, oc = (T + 127) / 128;
    t.tokens = (int)(128 / G);
    t.seq_streams = Tq <= t.tokens;
    t.seq_tiles = (int)((Tq + 2 * t.tokens - 1) / (2 * t.tokens));
    const int64_t seq = B * Hkv * t.seq_tiles;
    t.joint = P > 0 && rows * 4 >= (int64_t)t.seq_tiles * 256 * 3;
    if (t.joint) {
        // whole rounds of one tile an SM are not split (no parts to write, read and join); the tiles
        // of the last, short round are, so that it too fills the GPU
        t.whole = (int)(seq / kSMs * kSMs);
        const int64_t rest = seq - t.whole;
        p.So = rest ? balance(rest, pc + oc, 4, kSMs, most_splits(rest)) : 1;
        if (p.So == 1) t.whole = (int)seq;
        if (t.whole) p.part_rows = (seq - t.whole) * 256;
        p.merge = p.So > 1;
        p.parts_o = p.merge ? p.So : 0;
        t.seq_items = (int)(t.whole + (seq - t.whole) * p.So);
        return p;
    }
    double beside = 0;  // the few-row kernel's work on the own caches, in chunks of the tensor-core kernel a SM
    // Few rows: the few-row kernel reads the keys once for each 16 of them, from L2 after the first
    // time, where the tensor-core kernel reads them once but has a fixed cost of some 6 us (20 rows:
    // 12.4 against 13.7 us at 17 MB of keys, 26 against 22 at 67 MB). With scores that cost comes
    // twice, and a few rows' logits are cheap (20 rows: 20 / 33 / 66 us against 23 / 34 / 81 at 17 /
    // 67 / 268 MB; 32 rows: 32 against 26 at 33 MB).
    const int64_t tiles = (rows + kFewRows - 1) / kFewRows, again = (tiles - 1) * B * T * Hkv * D * 4;
    if (tiles == 1 || (rows <= kMostFew && (again <= 16 << 20 || (scored && rows <= 24)))) {
        p.rows.own_tiles = (int)tiles;
        p.parts_o = p.So = few_splits(B * Hkv * tiles, (T + 63) / 64, B > 1);
        p.rows.own_items = (int)(B * Hkv * tiles * p.So);
        // about 6 MB of keys a microsecond, caches three quarters full; a chunk takes 1.6 us
        beside = 0.75 * (double)(B * T * Hkv * D * 4) / 6e6 / 1.6;
        p.rows.pitch = (T + 15) / 16 * 16;
        p.logits = scored;
    } else {
        p.So = balance(seq, t.seq_streams ? (oc + 1) / 2 : oc, 4, kSMs, most_splits(seq));
        p.parts_o = p.So * (t.seq_streams ? 2 : 1);
        t.seq_items = (int)(seq * p.So);
    }
    if (B * rows <= kFewRows) {
        p.parts_p = p.Sp = few_splits(Hkv, (P + 63) / 64, false);
        p.rows.prefix_items = (int)(Hkv * p.Sp);
    } else {
        t.batch_streams = B * Tq <= t.tokens;
        t.batch_tiles = (int)((B * Tq + 2 * t.tokens - 1) / (2 * t.tokens));
        const int64_t batch = (int64_t)Hkv * t.batch_tiles;
        p.Sp = balance_beside(batch, t.batch_streams ? (pc + 1) / 2 : pc, 4, kSMs, beside, most_splits(batch));
        p.parts_p = p.Sp * (t.batch_streams ? 2 : 1);
        t.batch_items = (int)(Hkv * t.batch_tiles * p.Sp);
        p.rows.follows = t.batch_items > 0;
    }
    return p;
}

bool sizes_ok(int64_t B, int64_t Tq, int64_t Hq, int64_t Hkv, int64_t D, int64_t P, int64_t T) {
    if (B < 0 || Tq < 0 || P < 0 || T < 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || Hq / Hkv > 64) return false;
    if (D != 64 && D != 128) return false;
    // rows, work items and keys are counted in 32 bits (offsets in 64)
    if (B > (1 << 24) / Hkv || Hkv > 1 << 16) return false;
    return P <= INT32_MAX - 256 && T <= INT32_MAX - 256 && B <= INT32_MAX && Tq <= INT32_MAX && Hq <= INT32_MAX &&
           (B == 0 || Tq == 0 || B * Tq <= INT32_MAX / Hq);
}

int64_t round256(int64_t x) { return (x + 255) / 256 * 256; }

constexpr int64_t kWaitNs = 1000000000;
std::atomic<int64_t> g_wait_ns{kWaitNs};

}  // namespace

uint64_t wait_limit_ns() { return (uint64_t)g_wait_ns.load(std::memory_order_relaxed); }

int launch_prefix_finish(const PrefixArgs& a, const TilePlan& tp, int dtype, int D, const RowsPlan& rp,
                         const float* scores, float* scores_out, cudaStream_t stream) {
    if (dtype == kF32) return finish_d<float>(a, tp, D, rp, scores, scores_out, stream);
    if (dtype == kF16) return finish_d<__half>(a, tp, D, rp, scores, scores_out, stream);
    return finish_d<__nv_bfloat16>(a, tp, D, rp, scores, scores_out, stream);
}

}  // namespace lsa

using namespace lsa;

extern "C" {

int64_t lsa_shared_prefix_scratch(int dtype, int64_t B, int64_t Tq, int64_t Hq, int64_t Hkv, int64_t D, int64_t P,
                                  int64_t T, int scored) {
    if (!sizes_ok(B, Tq, Hq, Hkv, D, P, T) || dtype < kF32 || dtype > kBF16) return LSA_ERR_ARG;
    if (B == 0 || Tq == 0) return 0;
    const Plan p = make_plan(dtype, B, Tq, Hkv, Hq / Hkv, D, P, T, scored);
    const int64_t rows = B * Tq * Hq;
    const int64_t parts = p.parts_p + p.parts_o;
    return round256(parts * p.part_rows * D * 4) + round256(parts * p.part_rows * 4) + round256(rows * 4) +
           (p.logits ? round256(rows * p.rows.pitch * 4) : 0);
}

int lsa_shared_prefix_wait_limit(int64_t limit_ns) {
    if (limit_ns > 10 * kWaitNs) return LSA_ERR_ARG;
    g_wait_ns.store(limit_ns < 0 ? kWaitNs : limit_ns, std::memory_order_relaxed);
    return LSA_OK;
}

int lsa_shared_prefix_attention(const void* q, const void* k_prefix, const void* v_prefix, const void* k,
                                const void* v, int dtype, const int64_t* strides, const int32_t* lengths, int64_t B,
                                int64_t Tq, int64_t Hq, int64_t Hkv, int64_t D, int64_t P, int64_t T, float scale,
                                void* out, float* lse, const float* scores, float* scores_out, void* scratch,
                                int64_t scratch_bytes, int32_t* status, cudaStream_t stream) {
    if (!sizes_ok(B, Tq, Hq, Hkv, D, P, T) || dtype < kF32 || dtype > kBF16) return LSA_ERR_ARG;
    if ((scores == nullptr) != (scores_out == nullptr) || strides == nullptr) return LSA_ERR_ARG;
    const float scale_log2 = scale * 1.4426950408889634f;
    if (!(scale_log2 > 0.0f) || !(scale_log2 < INFINITY)) return LSA_ERR_ARG;  // the kernels take the maximum before it
    if (B == 0 || Tq == 0) {  // no row: the scores are what they were
        if (B == 0 || T == 0 || scores_out == scores) return LSA_OK;
        return cudaMemcpyAsync(scores_out, scores, (size_t)(B * Hkv * T) * 4, cudaMemcpyDeviceToDevice, stream) ==
                       cudaSuccess
                   ? LSA_OK
                   : LSA_ERR_CUDA;
    }
    if (q == nullptr || out == nullptr || lengths == nullptr || scratch == nullptr || status == nullptr) return LSA_ERR_ARG;
    if ((P > 0 && (k_prefix == nullptr || v_prefix == nullptr)) || (T > 0 && (k == nullptr || v == nullptr)))
        return LSA_ERR_ARG;
    // 16-byte loads: every base and every stride
    const int64_t unit = dtype == kF32 ? 4 : 8;
    for (const void* p : {q, P ? k_prefix : nullptr, P ? v_prefix : nullptr, T ? k : nullptr, T ? v : nullptr,
                          (const void*)out, (const void*)scratch})
        if ((uintptr_t)p & 15) return LSA_ERR_ARG;
    // a dimension of one entry takes any stride: D stands for it
    const int64_t ph = P ? Hkv : 1, ob = T ? B : 1, oh = T ? Hkv : 1;  // nor do the strides of nothing matter
    const int64_t extent[13] = {B, Tq, Hq, P, ph, P, ph, ob, T, oh, ob, T, oh};
    int64_t st[13];
    for (int i = 0; i < 13; ++i) {
        st[i] = extent[i] > 1 ? strides[i] : D;
        if (st[i] <= 0 || st[i] % unit || st[i] >= (int64_t)1 << 38) return LSA_ERR_ARG;
    }
    // the tensor-core kernel's tiles run over all sequences' tokens: one stride between them
    if (dtype != kF32 && B > 1 && Tq > 1 && st[0] != Tq * st[1]) return LSA_ERR_ARG;
    if (scratch_bytes < lsa_shared_prefix_scratch(dtype, B, Tq, Hq, Hkv, D, P, T, scores != nullptr)) return LSA_ERR_ARG;
    const Plan p = make_plan(dtype, B, Tq, Hkv, Hq / Hkv, D, P, T, scores != nullptr);
    PrefixArgs a;
    a.q = q, a.kp = k_prefix, a.vp = v_prefix, a.k = k, a.v = v;
    a.q_b = st[0], a.q_t = st[1], a.q_h = st[2];
    a.kp_t = st[3], a.kp_h = st[4], a.vp_t = st[5], a.vp_h = st[6];
    a.k_b = st[7], a.k_t = st[8], a.k_h = st[9];
    a.v_b = st[10], a.v_t = st[11], a.v_h = st[12];
    a.lengths = lengths;
    a.out = out;
    a.lse = lse;
    a.B = (int)B, a.Tq = (int)Tq, a.Hq = (int)Hq, a.Hkv = (int)Hkv, a.G = (int)(Hq / Hkv);
    a.P = (int)P, a.T = (int)T;
    a.Sp = p.Sp, a.So = p.So, a.parts_p = p.parts_p, a.parts_o = p.parts_o;
    a.status = status;
    a.wait_ns = wait_limit_ns();
    a.rows = B * Tq * Hq;
    a.part_rows = p.part_rows;
    a.scale_log2 = scale_log2;
    uint8_t* s = static_cast<uint8_t*>(scratch);
    a.part_o = reinterpret_cast<float*>(s);
    s += round256((p.parts_p + p.parts_o) * a.part_rows * D * 4);
    a.part_lse = reinterpret_cast<float*>(s);
    s += round256((p.parts_p + p.parts_o) * a.part_rows * 4);
    a.lse2 = reinterpret_cast<float*>(s);
    RowsPlan few = p.rows;
    if (p.logits && T > 0) few.logits = reinterpret_cast<float*>(s + round256(a.rows * 4));
    int rc = LSA_OK;
    if (p.simt) {
        rc = launch_prefix_simt(a, (int)D, stream);
    } else {
        rc = launch_prefix_tiles(a, p.tile, dtype, (int)D, stream);
        if (rc == LSA_OK) rc = launch_prefix_rows(a, few, dtype, (int)D, stream);
    }
    if (rc == LSA_OK && p.merge)
        rc = launch_prefix_finish(a, p.tile, dtype, (int)D, few, scores, scores_out, stream);
    if (rc == LSA_OK && scores && T > 0 && !p.logits)
        rc = p.simt ? launch_own_weights(a, (int)D, scores, scores_out, stream)
                    : launch_tile_weights(a, dtype, (int)D, scores, scores_out, stream);
    return rc;
}

}  // extern "C"
