// scored_tile.cu - attention weights of the own keys for many rows, on the tensor cores (sm_100a).
//
// With the rows' lse known, key j gains w_j = sum_r 2^(s_rj - lse_r). The scores are computed
// again, transposed: S^T = K Q^T with M = 128 keys and N = 128 rows, so a key is a TMEM lane, one
// thread holds it, and the sum over the rows never leaves the thread (no reduction, one order, one
// writer). K is read a second time, 256 bytes a key and head against the 512 r bytes that keeping
// the logits of r rows would move. A CTA walks pairs of key tiles of one (sequence, KV head); the
// two epilogue warpgroups own a tile of the pair each, with two S^T buffers of 128 TMEM columns
// apiece. Row tiles are whole tokens ((token, query head of the group) rows, 128 / G tokens); up
// to two of them stay in shared memory, more are streamed once per pair.
// What bounds it: the memory and the exponential units about alike (128 rows: 2048 cycles of exponentials
// a pair of tiles, 2900 in all). 32 rows x 4 heads of 4 sequences of 24576 keys: 41 us = 4.9 TB/s of K
// (the kernel alone). Fewer rows take the same: a tile's 128 columns are walked whatever is live (8 rows x 4 heads of 4
// ragged sequences of up to 32768 keys, both passes: 134 us called in a loop, 32 rows: 141).
// Warps: 0 TMA loads, 1 MMAs, 4-7 / 8-11 epilogue of the pair's first / second tile. What keys at
// or past a sequence's length hold stays in their own lanes, which store nothing but the old score.
#include "prefix_umma.cuh"

namespace lsa {
namespace {

constexpr int kThreads = 384;
constexpr int kKStages = 4;
constexpr int kQStages = 2;

struct WeightMaps {
    CUtensorMap k, q;
};

struct WeightPlan {
    int splits;     // of a (sequence, KV head)'s key pairs
    int row_tiles;  // of a sequence
    int tokens;     // of a row tile
};

template <int D> struct WeightShape {
    static constexpr int kTileBytes = kChunk * D * 2;
    static constexpr int kOffQ = kKStages * kTileBytes;
    static constexpr int kOffLse = kOffQ + kQStages * kTileBytes;  // [2 groups][2][128] fp32
    static constexpr int kOffBar = kOffLse + 4 * 128 * 4;
    static constexpr int kNumBars = 2 * kKStages + 2 * kQStages + 8 + 1;
    static constexpr int kOffMisc = kOffBar + kNumBars * 8;
    static constexpr int kSmem = kOffMisc + 16 + 1024;
    static_assert(kSmem <= 232448, "shared memory of a CTA");
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    weights_tile_kernel(const __grid_constant__ WeightMaps maps, const PrefixArgs a, const WeightPlan wp,
                        const float* __restrict__ scores, float* __restrict__ scores_out) {
    using Sh = WeightShape<D>;
    extern __shared__ uint8_t raw[];
    uint8_t* sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(sm);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Sh::kOffBar);
    uint64_t *kfull = bars, *kempty = kfull + kKStages, *qfull = kempty + kKStages, *qempty = qfull + kQStages,
             *sfull = qempty + kQStages, *sfree = sfull + 4, *drain = sfree + 4;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + Sh::kOffMisc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + Sh::kOffMisc + 4);
    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    grid_wait();
    grid_trigger();
    int i = blockIdx.x;
    const int split = i % wp.splits;
    i /= wp.splits;
    const int h = i % a.Hkv, b = i / a.Hkv;
    const int len = own_length(a, b);
    const int pairs = (int)(((int64_t)len + 2 * kChunk - 1) / (2 * kChunk));
    const int p0 = (int)((int64_t)pairs * split / wp.splits), p1 = (int)((int64_t)pairs * (split + 1) / wp.splits);
    const int nr = wp.row_tiles, tile_rows = wp.tokens * a.G;
    const bool resident = nr <= kQStages;
    const int64_t bh = ((int64_t)b * a.Hkv + h) * a.T;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kKStages; ++s) mbar_init(&kfull[s], 1), mbar_init(&kempty[s], 1);
        for (int s = 0; s < kQStages; ++s) mbar_init(&qfull[s], 1), mbar_init(&qempty[s], 1);
        for (int s = 0; s < 4; ++s) mbar_init(&sfull[s], 1), mbar_init(&sfree[s], 128);
        mbar_init(drain, 1);
        *abort_flag = a.wait_ns == 0;  // then the MMA thread gives up before its first wait, copies in flight
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) tmem_alloc(tmem_slot, 512);
    // rows of a Q stage that no box fills (128 is not a multiple of G): zeros, so their scores are
    for (int s = 0; s < kQStages * (D / 64); ++s)
        for (int r = tile_rows * 8 + threadIdx.x; r < 128 * 8; r += kThreads)
            *reinterpret_cast<uint4*>(sm + Sh::kOffQ + s * 16384 + r * 16) = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        // ---------------------------------------------------- loads
        int kpos = 0, qpos = 0;
        auto load_k = [&](int t) -> bool {
            const int s = kpos % kKStages;
            if (kpos >= kKStages && !role_wait(&kempty[s], (kpos / kKStages - 1) & 1, abort_flag, a.wait_ns)) return false;
            if (lane == 0) {
                mbar_arrive_expect_tx(&kfull[s], Sh::kTileBytes);
#pragma unroll
                for (int x = 0; x < D; x += 64)
                    tma_tile(sbase + s * Sh::kTileBytes + x * 256, &maps.k, x, t * kChunk, h, b, &kfull[s]);
            }
            __syncwarp();
            ++kpos;
            return true;
        };
        auto load_q = [&](int t) -> bool {
            const int s = qpos % kQStages;
            if (qpos >= kQStages && !role_wait(&qempty[s], (qpos / kQStages - 1) & 1, abort_flag, a.wait_ns)) return false;
            if (lane == 0) {
                mbar_arrive_expect_tx(&qfull[s], tile_rows * D * 2);
#pragma unroll
                for (int x = 0; x < D; x += 64)
                    tma_tile(sbase + Sh::kOffQ + s * Sh::kTileBytes + x * 256, &maps.q, x, h * a.G, t * wp.tokens, b,
                             &qfull[s]);
            }
            __syncwarp();
            ++qpos;
            return true;
        };
        bool ok = true;
        if (resident && p0 < p1)
            for (int t = 0; t < nr; ++t) load_q(t);
        for (int p = p0; ok && p < p1; ++p) {
            const int q = p0 + p1 - 1 - p;  // from the end: what the attention pass read last is still in L2
            ok = load_k(2 * q) && load_k(2 * q + 1);
            if (!resident)
                for (int t = 0; ok && t < nr; ++t) ok = load_q(t);
        }
        // every copy issued lands before the CTA leaves, whichever role gave up
        for (int p = kpos > kKStages ? kpos - kKStages : 0; p < kpos; ++p)
            mbar_wait_bounded(&kfull[p % kKStages], (p / kKStages) & 1);
        for (int p = qpos > kQStages ? qpos - kQStages : 0; p < qpos; ++p)
            mbar_wait_bounded(&qfull[p % kQStages], (p / kQStages) & 1);
    } else if (warp == 1) {
        // ---------------------------------------------------- MMAs
        constexpr uint32_t idS = umma_idesc_f16<T>(128, 128, false);
        if (elect_one()) {
            const uint64_t kd0 = sw128_desc(sbase, 16, 1024), qd0 = sw128_desc(sbase + Sh::kOffQ, 16, 1024);
            int kpos = 0, qpos = 0, it = 0;
            bool ok = *abort_flag == 0;
            for (int p = p0; ok && p < p1; ++p, kpos += 2) {
                for (int t = 0; ok && t < nr; ++t, ++it) {
                    const int q = resident ? t : qpos;
                    ok = thread_wait(&qfull[q % kQStages], resident ? 0 : (q / kQStages) & 1, abort_flag, a.wait_ns);
                    for (int g = 0; ok && g < 2; ++g) {
                        const int ks = (kpos + g) % kKStages, buf = 2 * g + (it & 1);
                        if (t == 0) ok = thread_wait(&kfull[ks], ((kpos + g) / kKStages) & 1, abort_flag, a.wait_ns);
                        if (ok && it >= 2) ok = thread_wait(&sfree[buf], (it / 2 - 1) & 1, abort_flag, a.wait_ns);
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t kd = desc_at(kd0, ks * Sh::kTileBytes);
                        const uint64_t qd = desc_at(qd0, (q % kQStages) * Sh::kTileBytes);
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk) {
                            const uint32_t off = (kk >> 2) * 16384 + (kk & 3) * 32;
                            umma_f16_ss(tmem + buf * 128, desc_at(kd, off), desc_at(qd, off), idS, kk > 0);
                        }
                        umma_commit(&sfull[buf]);
                        if (t == nr - 1) umma_commit(&kempty[ks]);
                        if (g == 1 && !resident) umma_commit(&qempty[q % kQStages]);
                    }
                    ++qpos;
                }
            }
            umma_commit(drain);  // every MMA completes before the TMEM is released
            mbar_wait_bounded(drain, 0);
        }
        __syncwarp();
    } else if (warp >= 4) {
        // ---------------------------------------------------- weights: group g, tile 2p + g
        const int g = (warp - 4) >> 2, tid = threadIdx.x & 127;
        float* nlse = reinterpret_cast<float*>(sm + Sh::kOffLse) + g * 256;
        const int nrows = a.Tq * a.G;
        auto lse_of = [&](int t) -> float {  // of row `tid` of row tile t; -inf weighs nothing
            const int r = t * tile_rows + tid;
            if (tid >= tile_rows || r >= nrows) return -INFINITY;
            const int tok = r / a.G;
            const float x = a.lse2[row_index(a, (int64_t)b * a.Tq + tok, h, r - tok * a.G)];
            return x == -INFINITY ? -INFINITY : -x;  // such a row sees no key
        };
        auto group_sync = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory"); };
        // the entries past the sequence's keys keep their scores
        int e0, e1;
        split_range(a.T - len, split, wp.splits, 1, &e0, &e1);
        for (int j = len + e0 + (int)threadIdx.x - 128; j < len + e1; j += 256) scores_out[bh + j] = scores[bh + j];
        if (resident && p0 < p1) {
            for (int t = 0; t < nr; ++t) nlse[t * 128 + tid] = lse_of(t);
            group_sync();
        }
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint64_t sl2 = pair(a.scale_log2, a.scale_log2);
        bool ok = true;
        int it = 0;
        for (int p = p0; p < p1; ++p) {  // to the end also after an expired wait: the group's barriers pair up
            const int j = (2 * (p0 + p1 - 1 - p) + g) * kChunk + tid;
            const float old = j < len ? scores[bh + j] : 0.0f;
            // rows before this one do not see key j
            const int64_t first = ((int64_t)j - (len - a.Tq)) * a.G;
            uint64_t sum[4] = {0ull, 0ull, 0ull, 0ull};
            for (int t = 0; t < nr; ++t, ++it) {
                const int buf = 2 * g + (it & 1);
                const float* nl = nlse + (resident ? t : it & 1) * 128;
                if (!resident) {
                    nlse[(it & 1) * 128 + tid] = lse_of(t);
                    group_sync();  // also: the buffer of two iterations ago has been read
                }
                ok = ok && role_wait(&sfull[buf], (it >> 1) & 1, abort_flag, a.wait_ns);
                if (!ok) continue;
                tc_fence_after();
                const int64_t before = first - (int64_t)t * tile_rows;  // keys x heads: past 32 bits either way
                const int hide = before > 128 ? 128 : (before < 0 ? 0 : (int)before);  // columns below it are hidden
                const bool masked = __any_sync(0xFFFFFFFFu, hide > 0);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t s[64];
                    tmem_ld64_wait<0>(tmem + lanes + buf * 128 + half * 64, s);
                    if (half == 1) {
                        tc_fence_before();
                        mbar_arrive(&sfree[buf]);
                    }
                    if (masked) {
#pragma unroll
                        for (int c = 0; c < 64; ++c)
                            if (half * 64 + c < hide) s[c] = 0xFF800000u;
                    }
#pragma unroll
                    for (int c = 0; c < 64; c += 4) {
                        const float4 n4 = *reinterpret_cast<const float4*>(nl + half * 64 + c);
                        float x0, x1, x2, x3;
                        unpair(fma2(pair(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), sl2, pair(n4.x, n4.y)), x0,
                               x1);
                        unpair(fma2(pair(__uint_as_float(s[c + 2]), __uint_as_float(s[c + 3])), sl2,
                                    pair(n4.z, n4.w)),
                               x2, x3);
                        sum[(c >> 1) & 3] = add2(sum[(c >> 1) & 3], pair(ex2_approx(x0), ex2_approx(x1)));
                        sum[((c >> 1) + 1) & 3] = add2(sum[((c >> 1) + 1) & 3], pair(ex2_approx(x2), ex2_approx(x3)));
                    }
                }
            }
            float x[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) unpair(sum[e], x[2 * e], x[2 * e + 1]);
            if (ok && j < len)
                scores_out[bh + j] = old + (((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7])));
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    if (threadIdx.x == 0 && *abort_flag) atomicExch(a.status, LSA_ERR_TIMEOUT);
}

template <typename T, int D>
int launch(const WeightMaps& maps, const PrefixArgs& a, const WeightPlan& wp, unsigned grid, const float* scores,
           float* scores_out, cudaStream_t stream) {
    if (!allow_kernel<weights_tile_kernel<T, D>>(WeightShape<D>::kSmem)) return LSA_ERR_CUDA;
    return launch_after(weights_tile_kernel<T, D>, dim3(grid), kThreads, WeightShape<D>::kSmem, stream, maps, a, wp,
                        scores, scores_out);
}

}  // namespace

int launch_tile_weights(const PrefixArgs& a, int dtype, int D, const float* scores, float* scores_out,
                        cudaStream_t stream) {
    if (encode_fn() == nullptr) return LSA_ERR_CUDA;
    WeightPlan wp;
    wp.tokens = 128 / a.G;
    wp.row_tiles = (a.Tq + wp.tokens - 1) / wp.tokens;
    // one CTA an SM: the splits that fill whole rounds best, each of at least two pairs of key tiles
    const int64_t units = (int64_t)a.B * a.Hkv, pairs = ((int64_t)a.T + 2 * kChunk - 1) / (2 * kChunk);
    wp.splits = balance(units, (pairs + 1) / 2, 2, 148, 4 * kMaxSplits);
    if (units * wp.splits > INT32_MAX) return LSA_ERR_SIZE;
    WeightMaps maps;
    const bool bf = dtype == kBF16;
    if (!encode_keys(&maps.k, bf, a.k, D, a.T, a.Hkv, a.B, a.k_t, a.k_h, a.k_b) ||
        !encode_map(&maps.q, bf, a.q, D, a.Hq, a.Tq, a.B, a.q_h, a.q_t, a.q_b, a.G, wp.tokens))
        return LSA_ERR_ARG;
    const unsigned grid = (unsigned)(units * wp.splits);
    if (dtype == kBF16)
        return D == 128 ? launch<__nv_bfloat16, 128>(maps, a, wp, grid, scores, scores_out, stream)
                        : launch<__nv_bfloat16, 64>(maps, a, wp, grid, scores, scores_out, stream);
    return D == 128 ? launch<__half, 128>(maps, a, wp, grid, scores, scores_out, stream)
                    : launch<__half, 64>(maps, a, wp, grid, scores, scores_out, stream);
}

}  // namespace lsa
