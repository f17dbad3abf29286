// prefix_tile.cu - the shared-prefix attention on the 5th-generation tensor cores (sm_100a).
//
// A work item is a tile of query rows of one KV head x a range of 128-key chunks. Row tiles:
//   batch tiles  rows of all sequences ((b, token, query head of the group)), prefix keys only:
//                the whole batch meets each prefix key once;
//   seq tiles    rows of one sequence, its own keys - after the prefix's, when the sequence's
//                rows fill a tile by themselves (joint: no parts to join then).
// One CTA per item, two halves of 128 rows (M = 128 each):
//   S_h = Q_h K^T   tcgen05.mma kind::f16, Q and K in 128B-swizzled shared memory, S in TMEM
//   softmax         one thread per row: S row from TMEM, running maximum and sum in fp32 (exp2
//                   domain; O is rescaled only when the maximum has grown by more than 2^kGrow), P
//                   back over S as 16-bit pairs
//   O_h += P_h V    tcgen05.mma with A = P from TMEM, V an MN-major shared-memory operand
// With more than 128 rows the halves are different rows of the same chunks; with at most 128 both
// halves hold the same rows and take alternate chunks (two streams), which keeps two softmax
// chains in flight where the keys' bandwidth, not arithmetic, is the bound.
// P is rounded to the inputs' 16-bit type for its product (the sum l adds the unrounded fp32
// values); everything else is fp32.
//
// Warps: 0 loads K and V tiles by TMA (cp.async.bulk.tensor, one ring of 128-key tiles in the
// order the MMAs use them), one thread of warp 1 issues every MMA (unrolled: 64 cycles per 128 x 128 x
// 16 MMA, the pipe's rate), 2 zeroes a sequence's V tail, 4-7 / 8-11 are the softmax of half 0 / 1. TMEM: S_0/P_0 [0, 128),
// S_1/P_1 [128, 256), O_0 [256, 256 + D), O_1 [384, 384 + D).
// What bounds it: with two halves of rows, the chain of a half - S (8 MMAs, 512 cycles), its softmax (about
// 1400 cycles to the first 96 keys' P, 2200 with the other half's exponentials beside it), the rest
// of P V - of which two run at a time: 3000 cycles a pair of chunks, where the MMAs alone take 2048; over
// seconds, the power limit (SM clock 1.55 GHz). 148 tiles on 4096 keys: tensor pipe 62 % active, 64 % of
// the exponential units. 64 tokens of 32 sequences on 10007 prefix keys (32 / 8 heads, D 128): 308 us =
// 1.13 PFLOP/s in bursts of 40 graph replays (68 % of the measured burst rate), 352 us = 0.99 PFLOP/s called
// in a loop (70 % of the sustained one). With two streams, the keys: 50 GB/s an SM, 6.4 TB/s while the
// ring runs. A tile's dead rows cost what live ones do: the softmax masks them, it does not skip them.
// Not kept: a part of the exponentials as polynomials on the FMA pipe (every 8th pair: no change, every
// 4th 3 % slower, every 2nd 15 %); a polling MMA thread in place of try_wait (no change).
// Rows of V at or past a sequence's length are zeroed in shared memory before their product, so
// whatever an unwritten slot holds (0 x NaN) stays out.
//
// Every wait is bounded (PrefixArgs::wait_ns, 1 s unless set); an expired wait raises a CTA-wide
// flag, every role leaves, copies and MMAs in flight are waited for (bounded), the TMEM is released
// and LSA_ERR_TIMEOUT lands in the status word.
#include "prefix_umma.cuh"

namespace lsa {
namespace {

constexpr int kThreads = 384;

// log2 of the factor that the weights carry into P and the sum, and of the growth of a row's maximum that is
// let stand: bf16 has fp32's exponents; fp16 holds nothing below 2^-25, so its weights are 2^7 times as large
// (2^-32 of the maximum is kept) and reach 2^11, which leaves 2^4 for the rounding of huge logits.
template <typename T> constexpr float kLift = 0.0f;
template <> constexpr float kLift<__half> = 7.0f;
template <typename T> constexpr float kGrow = 8.0f;
template <> constexpr float kGrow<__half> = 4.0f;

struct TileMaps {
    CUtensorMap kp, vp, k, v, q;
};

template <int D> struct TileShape {
    static constexpr int kTileBytes = kChunk * D * 2;  // one K, V or half-Q tile
    static constexpr int kStages = D == 128 ? 5 : 10;
    static constexpr int kOffStage = 2 * kTileBytes;
    static constexpr int kOffBar = kOffStage + kStages * kTileBytes;
    static constexpr int kNumBars = 2 * kStages + 1 + 2 + 4 + 2 + 1 + 2;
    static constexpr int kOffMisc = kOffBar + kNumBars * 8;
    static constexpr int kSmem = kOffMisc + 16 + 1024;  // slack: the base is aligned to 1024 B
    static_assert(kSmem <= 232448, "shared memory of a CTA");
};

// What a CTA works on.
struct Item {
    bool own, streams;  // seq tile; both halves hold the same rows
    bool direct;        // all of its rows' keys: it writes the output itself
    int b, h, part, len;
    int rest;        // which of the split seq tiles
    int t0, tokens;  // first token of the tile, tokens of the segment (all sequences' or one's)
    int np;      // prefix chunks of the item's chunk list
    int c0, c1;  // its chunks of the list [0, np + own chunks)
};

__device__ __forceinline__ Item item_of(const PrefixArgs& a, const TilePlan& t) {
    Item w;
    w.rest = 0;
    int i = blockIdx.x;
    w.own = i >= t.batch_items;
    int chunks, S, split, tile;
    if (!w.own) {
        S = a.Sp;
        split = i % S, i /= S;
        tile = i % t.batch_tiles;
        w.h = i / t.batch_tiles;
        w.b = 0;
        w.len = 0;
        w.streams = t.batch_streams;
        w.tokens = a.B * a.Tq;
        w.t0 = tile * 2 * t.tokens;
        w.np = chunks = (a.P + kChunk - 1) / kChunk;
        w.part = 0;
        w.direct = false;
    } else {
        i -= t.batch_items;
        w.direct = i < t.whole;
        S = w.direct ? 1 : a.So;
        split = w.direct ? 0 : (i - t.whole) % S;
        w.rest = w.direct ? 0 : (i - t.whole) / S;
        seq_tile(a, t, w.direct ? i : t.whole + w.rest, &w.b, &w.h, &tile);
        w.len = own_length(a, w.b);
        w.streams = t.seq_streams;
        w.tokens = a.Tq;
        w.t0 = tile * 2 * t.tokens;
        const int end = w.t0 + 2 * t.tokens < a.Tq ? w.t0 + 2 * t.tokens : a.Tq;
        int seen = w.len - a.Tq + end;  // own keys that the tile's last row sees
        seen = seen < 0 ? 0 : seen;
        w.np = t.joint ? (a.P + kChunk - 1) / kChunk : 0;
        chunks = w.np + (seen + kChunk - 1) / kChunk;
        w.part = t.joint ? 0 : a.parts_p;
    }
    w.part += split * (w.streams ? 2 : 1);
    split_range(chunks, split, S, 1, &w.c0, &w.c1);
    return w;
}

template <typename T, int D>
__device__ __forceinline__ void softmax_half(const PrefixArgs& a, const TilePlan& tp, const Item& w, uint64_t* bars,
                                             uint8_t* stage, volatile int* abort_flag, uint32_t tmem) {
    using Sh = TileShape<D>;
    uint64_t *bar_s = bars + 2 * Sh::kStages + 1, *bar_p = bar_s + 2, *bar_o = bar_p + 4;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int hf = (warp - 4) >> 2, qd = warp & 3;
    int tok, g;
    bool live = tile_row(a, tp, w.streams ? 0 : hf, qd * 32 + lane, &tok, &g);
    tok += w.t0;
    live = live && tok < w.tokens;
    // own keys the row sees; a prefix key is seen by all
    const int own_limit = !live ? 0 : (w.own ? w.len - a.Tq + tok + 1 : 0);
    const int pre_limit = live ? a.P : 0;
    const uint32_t lanes = (uint32_t)(qd * 32) << 16;
    const uint32_t tS = tmem + lanes + hf * 128;
    const uint32_t tO = tmem + lanes + 256 + hf * 128;
    const int step = w.streams ? 2 : 1, first = w.c0 + (w.streams ? hf : 0);
    const int n = w.c1 > first ? (w.c1 - first + step - 1) / step : 0;
    float m = -INFINITY, l = 0.0f;
    const float sl = a.scale_log2, thresh = fminf(kGrow<T> / sl, 1e30f);
    bool ok = true;
    auto publish = [&](uint64_t* bar) {  // this warp's P so far: one arrival a warp
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };
    for (int j = 0; j < n; ++j) {
        const int c = first + j * step;
        const int seen = c < w.np ? pre_limit - c * kChunk : own_limit - (c - w.np) * kChunk;
        ok = role_wait(&bar_s[hf], j & 1, abort_flag, a.wait_ns);
        if (!ok) break;
        tc_fence_after();
        uint32_t s[128];
        tmem_ld128_wait(tS, s);
        if (__any_sync(0xFFFFFFFFu, seen < kChunk)) {
#pragma unroll
            for (int i = 0; i < 128; ++i)
                if (i >= seen) s[i] = 0xFF800000u;  // -inf
        }
        // The exponentials start from the maximum of the chunks before, while this chunk's is
        // found beside them (a longest path of 64 dependent steps otherwise): fp32 and 16-bit P
        // carry a factor of up to 2^kGrow as well as 1. Only when the maximum has grown by more does
        // the warp take the new one, do the first 96 keys again and rescale O - always on a row's
        // first chunk.
        float alpha = 1.0f;
        bool grow = false;
        uint64_t sum[4];
        const uint64_t sl2 = pair(sl, sl);
        auto exps = [&](uint32_t& pk, int e, uint64_t neg2) {
            float x0, x1;
            unpair(fma2(pair(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), sl2, neg2), x0, x1);
            const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
            sum[(e >> 1) & 3] = add2(sum[(e >> 1) & 3], pair(p0, p1));
            pk = pack16(p0, p1, (T*)nullptr);
        };
        uint64_t neg2;
#pragma unroll 1
        for (bool again = false;; again = true) {
            const float neg = (m == -INFINITY ? 0.0f : -m * sl) + kLift<T>;
            neg2 = pair(neg, neg);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] = 0ull;
            uint32_t pk[32], pk2[16];
#pragma unroll
            for (int i = 0; i < 32; ++i) exps(pk[i], 2 * i, neg2);
            tmem_st32(tS, pk);
#pragma unroll
            for (int i = 0; i < 16; ++i) exps(pk2[i], 64 + 2 * i, neg2);
            tmem_st16(tS + 32, pk2);
            if (again) break;
            float mx4[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) mx4[i] = fmaxf(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]));
#pragma unroll
            for (int i = 8; i < 128; i += 8)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    mx4[e] = max3(mx4[e], __uint_as_float(s[i + 2 * e]), __uint_as_float(s[i + 2 * e + 1]));
            const float mx = max3(mx4[0], mx4[1], fmaxf(mx4[2], mx4[3]));
            grow = mx > m + thresh;
            if (!__any_sync(0xFFFFFFFFu, grow)) break;
            if (grow) {
                alpha = ex2_approx((m - mx) * sl);
                m = mx;
            }
            // O_h holds the earlier chunks' sum here (their products were issued before S_h(j) by
            // the same thread); its rescale lands before any P of this chunk is published
            if (j > 0) {
#pragma unroll 1
                for (int cc = 0; cc < D / 32; ++cc) {
                    uint32_t o[32];
                    tmem_ld32_wait(tO + cc * 32, o);
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                    tmem_st32(tO + cc * 32, o);
                }
            }
        }
        publish(&bar_p[2 * hf]);
        {
            uint32_t pk2[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) exps(pk2[i], 96 + 2 * i, neg2);
            tmem_st16(tS + 48, pk2);
        }
        publish(&bar_p[2 * hf + 1]);
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) unpair(sum[i], x[2 * i], x[2 * i + 1]);
        l = l * alpha + (((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7])));
    }
    if (ok && n > 0) ok = role_wait(&bar_o[hf], 0, abort_flag, a.wait_ns);
    if (!ok) return;
    const int64_t rid = row_index(a, (int64_t)w.b * a.Tq + tok, w.h, g);
    const bool none = l == 0.0f;  // the row has seen no key (a NaN logit makes l NaN, and the output)
    const float inv = none ? 0.0f : 1.0f / l;
    const float lse = none ? -INFINITY : m * sl + (log2f(l) - kLift<T>);
    const int64_t prow = tp.whole ? (int64_t)w.rest * 256 + hf * 128 + qd * 32 + lane : rid;
    const int64_t at = (int64_t)(w.part + (w.streams ? hf : 0)) * a.part_rows + prow;
    if (live) {
        if (w.direct) {
            a.lse2[rid] = lse;
            if (a.lse) a.lse[rid] = lse * 0.69314718055994531f;
        } else {
            a.part_lse[at] = lse;
        }
    }
    if (n == 0) {  // a part without a key is not read
        if (w.direct && live)
            for (int i = 0; i < D / 8; ++i)
                reinterpret_cast<uint4*>(static_cast<T*>(a.out) + rid * D)[i] = make_uint4(0, 0, 0, 0);
        return;
    }
    // The row through shared memory (the ring: every MMA is done) and out by one bulk copy: a thread
    // holds a whole row, so its own stores would touch 32 rows an instruction. Rows 16 bytes apart
    // from a multiple of 128: eight lanes' 16-byte stores fall into different banks.
    tc_fence_after();
    constexpr int kPitch = D * 4 + 16;
    uint8_t* line = stage + ((warp - 4) * 32 + lane) * kPitch;
#pragma unroll
    for (int cc = 0; cc < D / 32; ++cc) {
        uint32_t o[32];
        tmem_ld32_wait(tO + cc * 32, o);
        if (w.direct) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t u[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    u[e] = pack16(__uint_as_float(o[8 * i + 2 * e]) * inv, __uint_as_float(o[8 * i + 2 * e + 1]) * inv,
                                  (T*)nullptr);
                *reinterpret_cast<uint4*>(line + cc * 64 + i * 16) = make_uint4(u[0], u[1], u[2], u[3]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                *reinterpret_cast<float4*>(line + cc * 128 + i * 16) =
                    make_float4(__uint_as_float(o[4 * i]) * inv, __uint_as_float(o[4 * i + 1]) * inv,
                                __uint_as_float(o[4 * i + 2]) * inv, __uint_as_float(o[4 * i + 3]) * inv);
        }
    }
    fence_proxy_async_smem();
    if (live) {
        if (w.direct)
            bulk_s2g(static_cast<T*>(a.out) + rid * D, smem_u32(line), D * 2);
        else
            bulk_s2g(a.part_o + at * D, smem_u32(line), D * 4);
    }
    bulk_commit_wait();
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    prefix_tile_kernel(const __grid_constant__ TileMaps maps, const PrefixArgs a, const TilePlan tp) {
    using Sh = TileShape<D>;
    constexpr int NS = Sh::kStages, KS = D / 16;
    extern __shared__ uint8_t raw[];
    uint8_t* sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(sm);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Sh::kOffBar);
    uint64_t *full = bars, *empty = bars + NS, *bar_q = bars + 2 * NS, *bar_s = bar_q + 1, *bar_p = bar_s + 2,
             *bar_o = bar_p + 4, *bar_drain = bar_o + 2, *bar_tail = bar_drain + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + Sh::kOffMisc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + Sh::kOffMisc + 4);
    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (warp == 1) tmem_alloc(tmem_slot, 512);
    if (threadIdx.x == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(bar_q, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar_s[i], 1);
            mbar_init(&bar_p[2 * i], 4);
            mbar_init(&bar_p[2 * i + 1], 4);
            mbar_init(&bar_o[i], 1);
        }
        mbar_init(bar_drain, 1);
        mbar_init(bar_tail, 1);
        mbar_init(bar_tail + 1, 32);
        *abort_flag = a.wait_ns == 0;  // then the MMA thread gives up before its first wait, copies in flight
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    grid_wait();  // the inputs, the lengths among them, and the parts' last readers
    grid_trigger();
    const Item w = item_of(a, tp);
    const int n = w.c1 - w.c0;
    // the item's last chunk reaches past the sequence's keys
    const bool tail = n > 0 && w.c1 > w.np && (w.c1 - w.np) * kChunk > w.len;
    // Tile p of the ring, in the order the MMAs use them: one chunk's K (two, with two streams)
    // ahead of the first V, then V and the K that follows in turn.
    auto load = [&](int p) {
        int c, val;
        if (!w.streams) {
            val = p & 1, c = p >> 1;
        } else if (p < 2 && p < n) {
            val = 0, c = p;
        } else if (n == 1) {
            val = 1, c = 0;
        } else {
            const int i = p - 2;
            val = i >= 2 * (n - 2) || (i & 1) == 0;
            c = i >= 2 * (n - 2) ? i - (n - 2) : (i >> 1) + (val ? 0 : 2);
        }
        c += w.c0;
        const int s = p % NS;
        const uint32_t dst = sbase + Sh::kOffStage + s * Sh::kTileBytes;
        const bool pre = c < w.np;
        const CUtensorMap* map = pre ? (val ? &maps.vp : &maps.kp) : (val ? &maps.v : &maps.k);
        const int t = (pre ? c : c - w.np) * kChunk, b = pre ? 0 : w.b;
        mbar_arrive_expect_tx(&full[s], Sh::kTileBytes);
#pragma unroll
        for (int x = 0; x < D; x += 64) tma_tile(dst + x * 256, map, x, t, w.h, b, &full[s]);
    };
    const int early = 2 * n < NS ? 2 * n : NS;
    if (threadIdx.x == 0 && n > 0) {
        // Q: whole tokens, the rows of one KV head (a box past the segment's tokens holds other
        // sequences' rows or zeros; their lanes of S and O are no one's)
        const int halves = w.streams ? 1 : 2;
        mbar_arrive_expect_tx(bar_q, halves * tp.tokens * a.G * D * 2);
        for (int hf = 0; hf < halves; ++hf)
#pragma unroll
            for (int x = 0; x < D; x += 64)
                tma_tile(sbase + hf * Sh::kTileBytes + x * 256, &maps.q, x, w.h * a.G,
                         w.b * a.Tq + w.t0 + hf * tp.tokens, 0, bar_q);
        for (int p = 0; p < early; ++p) load(p);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp >= 4) {
        // 384 threads launch at 168 registers: 128 x 56 + 256 x 224 = 384 x 168
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;" ::: "memory");
        softmax_half<T, D>(a, tp, w, bars, sm + Sh::kOffStage, abort_flag, tmem);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;" ::: "memory");
        if (warp == 0) {
            // ------------------------------------------------ loads
            if (lane == 0) {
                int p = early;
                for (; p < 2 * n; ++p) {
                    if (!thread_wait(&empty[p % NS], (p / NS - 1) & 1, abort_flag, a.wait_ns)) break;
                    load(p);
                }
                // Every copy issued lands before the CTA leaves, also when it was another role that gave up.
                if (n > 0) mbar_wait_bounded(bar_q, 0);
                for (int i = p > NS ? p - NS : 0; i < p; ++i) mbar_wait_bounded(&full[i % NS], (i / NS) & 1);
            }
            __syncwarp();
        } else if (warp == 1) {
            // ------------------------------------------------ every MMA of the CTA, from one thread
            constexpr uint32_t idS = umma_idesc_f16<T>(128, 128, false);
            constexpr uint32_t idO = umma_idesc_f16<T>(128, D, true);
            if (elect_one()) {
                const uint64_t qd0 = sw128_desc(sbase, 16, 1024);
                const uint64_t kd0 = sw128_desc(sbase + Sh::kOffStage, 16, 1024);
                const uint64_t vd0 = sw128_desc(sbase + Sh::kOffStage, 16384, 1024);
                const uint32_t q1 = w.streams ? 0 : Sh::kTileBytes;
                int stage = 0, phase = 0;  // of the next tile of the ring
                auto advance = [&]() {
                    if (++stage == NS) stage = 0, phase ^= 1;
                };
                auto scores = [&](int hf, int st) {
                    const uint64_t qd = desc_at(qd0, hf ? q1 : 0), kd = desc_at(kd0, st * Sh::kTileBytes);
#pragma unroll
                    for (int kk = 0; kk < KS; ++kk) {
                        const uint32_t off = (kk >> 2) * 16384 + (kk & 3) * 32;
                        umma_f16_ss(tmem + hf * 128, desc_at(qd, off), desc_at(kd, off), idS, kk > 0);
                    }
                    umma_commit(&bar_s[hf]);
                };
                // P_h's first 96 and last 32 keys as they come; O_h starts afresh on a half's first chunk
                auto product = [&](int hf, int st, bool fresh, uint32_t parity) -> bool {
                    const uint64_t vd = desc_at(vd0, st * Sh::kTileBytes);
                    const uint32_t o = tmem + 256 + hf * 128, p = tmem + hf * 128;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        if (!thread_wait(&bar_p[2 * hf + half], parity, abort_flag, a.wait_ns)) return false;
                        tc_fence_after();
#pragma unroll
                        for (int kk = 6 * half; kk < 6 + 2 * half; ++kk)
                            umma_f16_ts(o, p + kk * 8, desc_at(vd, kk * 2048), idO, kk > 0 || !fresh);
                    }
                    return true;
                };
                // the V tile at the front of the ring; its rows past the sequence's keys zeroed
                auto value = [&](bool last) -> bool {
                    if (!thread_wait(&full[stage], phase, abort_flag, a.wait_ns)) return false;
                    if (last && tail) {
                        mbar_arrive(bar_tail);
                        if (!thread_wait(bar_tail + 1, 0, abort_flag, a.wait_ns)) return false;
                    }
                    return true;
                };
                auto key = [&]() -> bool {
                    const bool ok = thread_wait(&full[stage], phase, abort_flag, a.wait_ns);
                    tc_fence_after();
                    return ok;
                };
                bool ok = *abort_flag == 0 && (n == 0 || thread_wait(bar_q, 0, abort_flag, a.wait_ns));
                if (ok && n > 0 && !w.streams) {
                    ok = key();
                    if (ok) {
                        scores(0, stage), scores(1, stage);
                        umma_commit(&empty[stage]);
                        advance();
                    }
                    for (int j = 0; ok && j < n; ++j) {
                        const bool more = j + 1 < n;
                        const int sv = stage;
                        if (!(ok = value(!more))) break;
                        advance();
                        if (!(ok = product(0, sv, j == 0, j & 1))) break;
                        if (more) {
                            if (!(ok = key())) break;
                            scores(0, stage);
                        }
                        if (!(ok = product(1, sv, j == 0, j & 1))) break;
                        umma_commit(&empty[sv]);
                        if (more) {
                            scores(1, stage);
                            umma_commit(&empty[stage]);
                            advance();
                        }
                    }
                } else if (ok && n > 0) {
                    for (int c = 0; ok && c < n && c < 2; ++c) {
                        ok = key();
                        if (ok) {
                            scores(c, stage);
                            umma_commit(&empty[stage]);
                            advance();
                        }
                    }
                    for (int c = 0; ok && c < n; ++c) {
                        const int hf = c & 1;
                        if (!(ok = value(c + 1 == n))) break;
                        if (!(ok = product(hf, stage, c < 2, (c >> 1) & 1))) break;
                        umma_commit(&empty[stage]);
                        advance();
                        if (c + 2 < n) {
                            if (!(ok = key())) break;
                            scores(hf, stage);
                            umma_commit(&empty[stage]);
                            advance();
                        }
                    }
                }
                if (ok) umma_commit(&bar_o[0]), umma_commit(&bar_o[1]);
                umma_commit(bar_drain);  // every MMA completes before the TMEM is released
                mbar_wait_bounded(bar_drain, 0);
            }
            __syncwarp();
        } else if (warp == 2 && tail) {
            // ------------------------------------------------ the tail of a sequence's last V tile
            // (a wait as long as the item: the MMA thread has up to four a chunk of its own before it)
            if (role_wait(bar_tail, 0, abort_flag, a.wait_ns * (4 * (uint64_t)n + 8))) {
                uint8_t* va = sm + Sh::kOffStage + ((2 * n - 1) % NS) * Sh::kTileBytes;  // the last load
                for (int i = (w.len - (w.c1 - 1 - w.np) * kChunk) * 8 + lane; i < kChunk * 8; i += 32)
#pragma unroll
                    for (int x = 0; x < D / 64; ++x)
                        *reinterpret_cast<uint4*>(va + x * 16384 + i * 16) = make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
                mbar_arrive(bar_tail + 1);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    if (threadIdx.x == 0 && *abort_flag) atomicExch(a.status, LSA_ERR_TIMEOUT);
}

template <typename T, int D>
int launch(const TileMaps& maps, const PrefixArgs& a, const TilePlan& tp, unsigned grid, cudaStream_t stream) {
    if (!allow_kernel<prefix_tile_kernel<T, D>>(TileShape<D>::kSmem)) return LSA_ERR_CUDA;
    return launch_after(prefix_tile_kernel<T, D>, dim3(grid), kThreads, TileShape<D>::kSmem, stream, maps, a, tp);
}

}  // namespace

int launch_prefix_tiles(const PrefixArgs& a, const TilePlan& tp, int dtype, int D, cudaStream_t stream) {
    const int64_t items = (int64_t)tp.batch_items + tp.seq_items;
    if (items == 0) return LSA_OK;
    if (items > INT32_MAX) return LSA_ERR_SIZE;
    if (encode_fn() == nullptr) return LSA_ERR_CUDA;
    TileMaps maps;
    const bool bf = dtype == kBF16;
    // q's tokens of all sequences in one dimension (the entry point checks that they are)
    bool ok = encode_map(&maps.q, bf, a.q, D, a.Hq, (int64_t)a.B * a.Tq, 1, a.q_h, a.Tq > 1 ? a.q_t : a.q_b, D, a.G,
                         tp.tokens);
    if (ok && a.P > 0 && (tp.batch_items || tp.joint))
        ok = encode_keys(&maps.kp, bf, a.kp, D, a.P, a.Hkv, 1, a.kp_t, a.kp_h, (int64_t)D) &&
             encode_keys(&maps.vp, bf, a.vp, D, a.P, a.Hkv, 1, a.vp_t, a.vp_h, (int64_t)D);
    if (ok && a.T > 0 && tp.seq_items)
        ok = encode_keys(&maps.k, bf, a.k, D, a.T, a.Hkv, a.B, a.k_t, a.k_h, a.k_b) &&
             encode_keys(&maps.v, bf, a.v, D, a.T, a.Hkv, a.B, a.v_t, a.v_h, a.v_b);
    if (!ok) return LSA_ERR_ARG;
    const unsigned grid = (unsigned)items;
    if (dtype == kBF16)
        return D == 128 ? launch<__nv_bfloat16, 128>(maps, a, tp, grid, stream)
                        : launch<__nv_bfloat16, 64>(maps, a, tp, grid, stream);
    return D == 128 ? launch<__half, 128>(maps, a, tp, grid, stream)
                    : launch<__half, 64>(maps, a, tp, grid, stream);
}

}  // namespace lsa
