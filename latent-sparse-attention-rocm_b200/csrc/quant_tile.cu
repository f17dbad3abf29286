// quant_tile.cu - attention over the 8-bit paged cache for many rows, on the 5th-generation tensor cores (sm_100a).
// quant.cuh has the formulas.
//
// A work item is a tile of query rows of one (sequence, KV head) - two halves of 128 rows (tokens x the G query heads
// of the group) - x a range of 128-key chunks. One CTA an item:
//   S_h = Q_h K^T   tcgen05.mma kind::f16, Q and K as fp16 in 128B-swizzled shared memory, S in TMEM
//   softmax         one thread a row, maximum and sums in fp32, P back over S as pairs of halves
//   O_h += P_h V    tcgen05.mma with A = P from TMEM, V an MN-major shared-memory operand
// With at most 128 rows both halves hold the same rows and take alternate chunks, so that two softmax chains are in
// flight where the keys' bandwidth is the bound.
// The codes come as they are (bulk copies of a page's rows of a head, which are contiguous) into a ring of 8-bit tiles;
// two warps, and softmax warps that no row wants, make halves of them (exact) into a ring of operand tiles, zeros where
// there is no key, so what a page holds behind a sequence's last token never meets a product. Scales stay out of the
// tiles: 16 keys (64 on pages of 64 or 128) share theirs, so a row's logits are s * (ks * factor) + log2 vs with
// constants for them, and the sum takes 1 / vs once.
// bf16 rows of Q become fp16 by a power of two of their own, as in the few-row kernel. P is rounded to fp16 and
// carries 2^kLift; the maximum is let stand until it has grown by more than 2^kGrow.
//
// Warps: 0 asks for the codes and the scales, one thread of warp 1 issues every MMA, 2 and 3 convert, 4-7 / 8-11 are
// the softmax of half 0 / 1. TMEM: S_0/P_0 [0, 128), S_1/P_1 [128, 256), O_0 [256, 256 + D), O_1 [384, 384 + D).
//
// What bounds it (B200, 32 / 8 heads, D 128): with two halves of rows the chain of a half - softmax 2350 cycles, then its
// product and the next S 1100 - of which two run at a time: 3400 cycles a pair of chunks, where the MMAs take 2048 and the
// exponentials as many; 2 x 1024 tokens on 16384 keys 497-536 us = 0.99-1.07 PFLOP/s in a loop (70-76 % of the sustained
// rate), 494 us = 1.08 PFLOP/s in bursts. With two streams, converting: about 1000 cycles a tile for two warps (500 alone;
// shared memory and the ALU pipe are the softmax's and the MMAs' too), 32 tokens on 65536 keys 65 us = 2.1 TB/s. Not
// kept: four more converting warps (a thread's 128 logits want 146 registers), loads of the next codes before the
// stores of these (no change), S and P in steps of 64 keys with the next step's S issued ahead (573 us against 538: what
// a step costs a warp beside its exponentials - waits, TMEM loads and stores, barriers - comes twice as often).
//
// Every wait is bounded (QuantArgs::wait_ns); an expired wait raises a CTA-wide flag, every role leaves, copies and
// MMAs in flight are waited for (bounded), the TMEM is released and LSA_ERR_TIMEOUT lands in the status word.
#include <type_traits>

#include "prefix_umma.cuh"
#include "quant.cuh"

namespace lsa {
namespace {

constexpr int kThreads = 384;
constexpr float kLift = 7.0f, kGrow = 4.0f;
constexpr int kChunks = 8;  // chunks whose scales are kept: more than the rings and the softmax hold together
constexpr int kGroups = kChunk / 16;

template <int D> struct QuantTile {
    static constexpr int kOperand = kChunk * D * 2;  // an fp16 K, V or half-Q tile
    static constexpr int kCodes = kChunk * D;        // its codes
    // Operand tiles and tiles of codes. A tile of one half's rows has the other half of Q for two more.
    static constexpr int kOps = D == 128 ? 3 : 6, kStages = D == 128 ? 4 : 5, kMore = kOperand / kCodes;
    static constexpr int kOffOps = 2 * kOperand;
    static constexpr int kOffStage = kOffOps + kOps * kOperand;
    static constexpr int kOffScales = kOffStage + kStages * kCodes;  // [kChunks][kGroups] (ks, log2 vs, 1 / vs, rows)
    static constexpr int kOffFactor = kOffScales + kChunks * kGroups * 16;
    static constexpr int kOffBar = kOffFactor + 256 * 4;
    static constexpr int kNumBars = 2 * (kStages + kMore) + 2 * kOps + 2 + 4 + 2 + 1;
    static constexpr int kOffMisc = kOffBar + kNumBars * 8;
    static constexpr int kSmem = kOffMisc + 16;
    static __device__ __forceinline__ int codes_at(int s) {
        return s < kStages ? kOffStage + s * kCodes : kOperand + (s - kStages) * kCodes;
    }
    static_assert(kSmem <= 232448, "shared memory of a CTA");
    static_assert(kOffStage >= 256 * (D * 4 + 16), "the rows leave through Q and the operand ring");
};

// What a CTA works on.
struct Item {
    int b, h, split, rest, t0;
    bool direct;       // all of its rows' keys: it writes the output itself
    int length, keys;  // tokens of the sequence; those that the table has room for
    int c0, c1;        // its chunks
};

__device__ __forceinline__ Item item_of(const QuantArgs& a) {
    Item w;
    int i = blockIdx.x;
    w.direct = i < a.whole;
    w.split = w.direct ? 0 : (i - a.whole) % a.parts;
    w.rest = w.direct ? 0 : (i - a.whole) / a.parts;
    int tile;
    quant_tile_at(a, w.direct ? i : a.whole + w.rest, &w.b, &w.h, &tile);
    const int tokens = (a.streams ? 1 : 2) * a.tokens;
    w.t0 = tile * tokens;
    const int end = w.t0 + tokens < a.Tq ? w.t0 + tokens : a.Tq;
    w.length = max(a.lengths[w.b], 0);
    const int64_t room = (int64_t)a.M << a.shift;
    w.keys = w.length < room ? w.length : (int)room;
    int seen = w.length - a.Tq + end;  // keys that the tile's last row sees
    seen = seen < 0 ? 0 : (seen < w.keys ? seen : w.keys);
    const int64_t chunks = (seen + kChunk - 1) / kChunk, S = w.direct ? 1 : a.parts;
    w.c0 = (int)(chunks * w.split / S), w.c1 = (int)(chunks * (w.split + 1) / S);
    return w;
}

// Tile p of an item of n chunks, in the order the MMAs use them: one chunk's K (two, with two streams) ahead of the
// first V, then V and the K that follows in turn.
__device__ __forceinline__ void tile_of(int p, int n, bool streams, int* c, bool* value) {
    if (!streams) {
        *value = p & 1, *c = p >> 1;
    } else if (p < 2 && p < n) {
        *value = false, *c = p;
    } else if (n == 1) {
        *value = true, *c = 0;
    } else {
        const int i = p - 2;
        *value = i >= 2 * (n - 2) || (i & 1) == 0;
        *c = i >= 2 * (n - 2) ? i - (n - 2) : (i >> 1) + (*value ? 0 : 2);
    }
}

// Row rl of half hf: (token of the call, head of the group); false: no row there.
__device__ __forceinline__ bool row_at(const QuantArgs& a, const Item& w, int hf, int rl, int* tok, int* g) {
    const int tl = token_of(a, rl);
    *tok = w.t0 + (a.streams ? 0 : hf) * a.tokens + tl;
    *g = rl - tl * a.G;
    return tl < a.tokens && *tok < a.Tq;
}

__device__ __forceinline__ float4 lds_f4(uint32_t addr) {
    float4 r;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(r.x), "=f"(r.y), "=f"(r.z), "=f"(r.w)
                 : "r"(addr)
                 : "memory");
    return r;
}
__device__ __forceinline__ uint4 lds_u4(uint32_t addr) {
    uint4 r;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "r"(addr)
                 : "memory");
    return r;
}
__device__ __forceinline__ void sts_u4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Q's rows as fp16 in their operand tiles, and each row's factor.
template <typename T, int D>
__device__ __forceinline__ void load_q(const QuantArgs& a, const Item& w, uint8_t* sm) {
    using Sh = QuantTile<D>;
    constexpr int L = D / 8, RP = (kThreads - 32) / L;  // threads of a row, rows of a pass
    constexpr int PASSES = (256 + RP - 1) / RP;
    float* factor = reinterpret_cast<float*>(sm + Sh::kOffFactor);
    const int t = threadIdx.x - 32, lr = t / L, ch = t % L;  // all warps but the first
    const int halves = a.streams ? 1 : 2;
    uint4 raw[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int row = i * RP + lr, hf = row >> 7;
        raw[i] = make_uint4(0, 0, 0, 0);
        int tok, g;
        if (row < halves * 128 && row_at(a, w, hf, row & 127, &tok, &g))
            raw[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + w.b * a.q_b + tok * a.q_t +
                                                     (w.h * (int64_t)a.G + g) * a.q_h + ch * 8);
    }
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int row = i * RP + lr, hf = row >> 7, r = row & 127;
        uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        float f = a.scale_log2;
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, max(u[e] & 0x7FFFu, (u[e] >> 16) & 0x7FFFu));
#pragma unroll
        for (int off = L / 2; off >= 1; off >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, off));
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            const float by = half_factor(top, &f);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                u[e] = pack16(__uint_as_float(u[e] << 16) * by, __uint_as_float(u[e] & 0xFFFF0000u) * by, (__half*)nullptr);
        }
        if (infinite_row<T>(top)) f = kInfiniteRow, u[0] = u[1] = u[2] = u[3] = 0;
        if (row < halves * 128) {
            sts_u4(smem_u32(sm) + hf * Sh::kOperand + (ch >> 3) * 16384 + r * 128 + (((ch & 7) ^ (r & 7)) << 4), u[0], u[1],
                   u[2], u[3]);
            if (ch == 0) factor[row] = f;
        }
    }
}

// How many 16-key steps of P are handed over ahead of the others: half, where a step's constants are at hand (2 x 1024
// tokens on 16384 keys 494 us in bursts, with six 517; pages of 16 619 against 585, D 64 244 against 238).
template <int D, int GK> constexpr int kFirst = GK == 64 && D == 128 ? 4 : 6;

template <typename T, int D, int GK>
__device__ __forceinline__ void softmax_half(const QuantArgs& a, const Item& w, uint8_t* sm, uint64_t* bar_s, uint64_t* bar_p,
                                             uint64_t* bar_o, volatile int* abort_flag, uint32_t tmem) {
    using Sh = QuantTile<D>;
    constexpr int FIRST = kFirst<D, GK>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int hf = (warp - 4) >> 2, qd = warp & 3;
    int tok, g;
    const bool live = row_at(a, w, hf, qd * 32 + lane, &tok, &g);
    const int limit = live ? w.length - a.Tq + tok + 1 : 0;  // keys the row sees
    const float factor = reinterpret_cast<const float*>(sm + Sh::kOffFactor)[(a.streams ? 0 : hf) * 128 + qd * 32 + lane];
    const uint32_t lanes = (uint32_t)(qd * 32) << 16;
    const uint32_t tS = tmem + lanes + hf * 128;
    const uint32_t tO = tmem + lanes + 256 + hf * 128;
    const int step = a.streams ? 2 : 1, first = w.c0 + (a.streams ? hf : 0);
    const int n = w.c1 > first ? (w.c1 - first + step - 1) / step : 0;
    const float4* const scales = reinterpret_cast<const float4*>(sm + Sh::kOffScales);
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    auto publish = [&](uint64_t* bar) {  // this warp's P so far: one arrival a warp
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };
    for (int j = 0; j < n; ++j) {
        const int c = first + j * step;
        const int seen = limit - c * kChunk;
        ok = role_wait(&bar_s[hf], j & 1, abort_flag, a.wait_ns);
        if (!ok) break;
        tc_fence_after();
        const float4* const sc = scales + (c % kChunks) * kGroups;
        uint32_t s[128];
        tmem_ld128_wait(tS, s);
        if (__any_sync(0xFFFFFFFFu, seen < kChunk)) {
#pragma unroll
            for (int i = 0; i < 128; ++i)
                if (i >= seen) s[i] = 0xFF800000u;  // -inf
        }
        // The exponentials start from the maximum of the chunks before, while this chunk's is found beside them. Only
        // when it has grown by more than 2^kGrow does the warp take the new one, do the first keys again and rescale O
        // - always on a row's first chunk.
        float alpha = 1.0f;
        uint64_t sum;
        // logits from s, GK keys at a time: (multiplier, addend); the multiplier stays above 0, so that -inf does. Of 64
        // keys, they are held; of 16, read when their turn comes.
        constexpr int NG = kChunk / GK;
        float muls[GK == 64 ? NG : 1], adds[GK == 64 ? NG : 1], invs[GK == 64 ? NG : 1];
        if constexpr (GK == 64) {
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                const float4 k = sc[i * (GK / 16)];
                muls[i] = fmaxf(k.x * factor, 1e-30f), adds[i] = k.y, invs[i] = k.z;
            }
        }
        auto group = [&](int i, float* mul, float* add) {  // of 16 keys
            if constexpr (GK == 64) {
                *mul = muls[i / 4], *add = adds[i / 4];
                return invs[i / 4];
            } else {
                const float4 k = sc[i];
                *mul = fmaxf(k.x * factor, 1e-30f), *add = k.y;
                return k.z;
            }
        };
        auto exps = [&](auto& pk, int at, int i, float neg) {  // 16 keys
            float mul, add;
            const float inv = group(i, &mul, &add);
            const uint64_t mul2x = pair(mul, mul), add2x = pair(add + neg, add + neg);
            uint64_t part[2] = {0ull, 0ull};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float x0, x1;
                unpair(fma2(pair(__uint_as_float(s[16 * i + 2 * e]), __uint_as_float(s[16 * i + 2 * e + 1])), mul2x, add2x), x0, x1);
                const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
                part[e & 1] = add2(part[e & 1], pair(p0, p1));
                pk[at + e] = pack16(p0, p1, (__half*)nullptr);
            }
            sum = fma2(add2(part[0], part[1]), pair(inv, inv), sum);
        };
        float neg;
#pragma unroll 1
        for (bool again = false;; again = true) {
            neg = (m == -INFINITY ? 0.0f : -m) + kLift;
            sum = 0ull;
            uint32_t pk[32];
#pragma unroll
            for (int i = 0; i < 4; ++i) exps(pk, 8 * i, i, neg);
            tmem_st32(tS, pk);
            if constexpr (FIRST == 6) {
                uint32_t pk2[16];
#pragma unroll
                for (int i = 0; i < 2; ++i) exps(pk2, 8 * i, 4 + i, neg);
                tmem_st16(tS + 32, pk2);
            }
            if (again) break;
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                float mul, add, mg[4];
                group(i * (GK / 16), &mul, &add);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    mg[e] = fmaxf(__uint_as_float(s[GK * i + 2 * e]), __uint_as_float(s[GK * i + 2 * e + 1]));
#pragma unroll
                for (int e = 8; e < GK; e += 2)
                    mg[e / 2 & 3] = max3(mg[e / 2 & 3], __uint_as_float(s[GK * i + e]), __uint_as_float(s[GK * i + e + 1]));
                mx = fmaxf(mx, fmaf(max3(mg[0], mg[1], fmaxf(mg[2], mg[3])), mul, add));
            }
            const bool grow = mx > m + kGrow;
            if (!__any_sync(0xFFFFFFFFu, grow)) break;
            if (grow) {
                alpha = ex2_approx(m - mx);
                m = mx;
            }
            // O_h holds the earlier chunks' sum here (their products were issued before S_h(j) by the same thread); its
            // rescale lands before any P of this chunk is published
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
            uint32_t rest[8 * (kGroups - FIRST)];
#pragma unroll
            for (int i = 0; i < kGroups - FIRST; ++i) exps(rest, 8 * i, FIRST + i, neg);
            if constexpr (FIRST == 6)
                tmem_st16(tS + 48, rest);
            else
                tmem_st32(tS + 32, rest);
        }
        publish(&bar_p[2 * hf + 1]);
        float s0, s1;
        unpair(sum, s0, s1);
        l = l * alpha + (s0 + s1);
    }
    if (ok && n > 0) ok = role_wait(&bar_o[hf], 0, abort_flag, a.wait_ns);
    if (!ok) return;
    const int64_t rid = ((int64_t)w.b * a.Tq + tok) * a.Hq + (int64_t)w.h * a.G + g;
    l = sum_of_row(l, factor);
    const bool none = l == 0.0f;  // the row has seen no key (a NaN makes the output NaN)
    const float inv = none ? 0.0f : 1.0f / l;
    const float lse = none ? -INFINITY : m + (log2f(l) - kLift);
    const int64_t at = quant_part_row(a, w.split, w.rest, hf, qd * 32 + lane);
    if (live) {
        if (!w.direct)
            a.part_lse[at] = lse;
        else if (a.lse)
            a.lse[rid] = lse * 0.69314718055994531f;
    }
    if (n == 0) {  // a part without a key is not read
        if (w.direct && live)
            for (int i = 0; i < D / 8; ++i)
                reinterpret_cast<uint4*>(static_cast<T*>(a.out) + rid * D)[i] = make_uint4(0, 0, 0, 0);
        return;
    }
    // The row through shared memory (every MMA is done) and out by one bulk copy: a thread holds a whole row, so its own
    // stores would touch 32 rows an instruction. Rows 16 bytes apart from a multiple of 128: eight lanes' 16-byte stores
    // fall into different banks.
    tc_fence_after();
    constexpr int kPitch = D * 4 + 16;
    uint8_t* line = sm + ((warp - 4) * 32 + lane) * kPitch;
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

// The warp that asks for codes and scales: a lane 16 keys of the chunk (whose page's rows the first lane of a page asks
// for), page ids two chunks ahead, scales one.
template <int D> struct Loader {
    using Sh = QuantTile<D>;
    int id0, id1, held[3];  // page ids of the next K's chunk and of the one after it; of the chunks whose V is to come
    float ks, vs;           // the next K's chunk's scales

    // page id of this lane's keys of the item's chunk c, -1: none
    static __device__ __forceinline__ int lookup(const QuantArgs& a, const Item& w, int c) {
        const int lane = threadIdx.x & 31;
        const int64_t key = (int64_t)(w.c0 + c) * kChunk + lane * 16;
        int id = -1;
        if (lane < kGroups && c < w.c1 - w.c0 && key < w.keys) id = a.table[w.b * a.table_ld + (key >> a.shift)];
        return id >= 0 && id < a.pages ? id : -1;
    }
    __device__ __forceinline__ void scales(const QuantArgs& a, const Item& w) {
        const int64_t head = (int64_t)(id0 < 0 ? 0 : id0) * a.Hkv + w.h;
        ks = id0 < 0 ? 1.0f : a.ks[head];
        vs = id0 < 0 ? 1.0f : a.vs[head];
    }
    __device__ __forceinline__ void start(const QuantArgs& a, const Item& w) {
        id0 = lookup(a, w, 0), id1 = lookup(a, w, 1);
        held[0] = held[1] = held[2] = -1;
        scales(a, w);
    }
    // Tile p into stage s.
    __device__ __forceinline__ void load(const QuantArgs& a, const Item& w, uint8_t* sm, uint64_t* codes_full, int p, int s) {
        const int lane = threadIdx.x & 31, page = 1 << a.shift;
        int c;
        bool value;
        tile_of(p, w.c1 - w.c0, a.streams, &c, &value);
        const int id = !value ? id0 : (c % 3 == 0 ? held[0] : (c % 3 == 1 ? held[1] : held[2]));
        const int left = id < 0 ? 0 : w.keys - (w.c0 + c) * kChunk - lane * 16;  // keys from the lane's first on
        const int rows = left < 0 ? 0 : (left < 16 ? left : 16);
        int total = rows;
#pragma unroll
        for (int off = 1; off < 8; off <<= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, off);
        if (lane == 0) mbar_arrive_expect_tx(&codes_full[s], total * D);
        __syncwarp();
        const int64_t head = (int64_t)(id < 0 ? 0 : id) * a.Hkv + w.h;
        if (rows > 0 && ((lane * 16) & (page - 1)) == 0)
            bulk_g2s(sm + Sh::codes_at(s) + lane * 16 * D, (value ? a.v8 : a.k8) + (head << a.shift) * D,
                     (left < page ? left : page) * D, &codes_full[s]);
        if (!value) {
            held[2] = c % 3 == 2 ? id : held[2], held[1] = c % 3 == 1 ? id : held[1], held[0] = c % 3 == 0 ? id : held[0];
            if (lane < kGroups) {
                const float v = fmaxf(vs, 8.6736174e-19f);  // 2^-60
                *reinterpret_cast<float4*>(sm + Sh::kOffScales + (((w.c0 + c) % kChunks) * kGroups + lane) * 16) =
                    rows > 0 ? make_float4(ks, log2f(v), 1.0f / v, __int_as_float(rows))
                             : make_float4(1.0f, -INFINITY, 0.0f, 0.0f);
            }
            __syncwarp();
            id0 = id1;
            scales(a, w);
            id1 = lookup(a, w, c + 2);
        }
        if (lane == 0) mbar_arrive(&codes_full[s]);
    }
};

// Codes to operand tiles: warp `self` of WARPS (even). A warp's step is 8 rows, four lanes a row, half of a row's 64-byte
// pieces each (D = 128: neighbouring rows at different blocks, so that both the loads and the stores miss each other's
// banks). Zeros where there is no key.
template <int CODE, int D, int WARPS>
__device__ __forceinline__ void convert(const QuantArgs& a, const Item& w, uint8_t* sm, uint64_t* codes_full,
                                        uint64_t* codes_empty, uint64_t* op_full, uint64_t* op_empty,
                                        volatile int* abort_flag, int self) {
    using Sh = QuantTile<D>;
    // Of two blocks, a warp takes the same one of all of its rows: steps first, first + BY .. of 8 rows
    constexpr int NO = Sh::kOps, X = D / 64, BY = WARPS / X, STEPS = (kChunk / 8 + BY - 1) / BY;
    const int NS = a.streams ? Sh::kStages + Sh::kMore : Sh::kStages;
    const int lane = threadIdx.x & 31, lr = lane >> 2, q = lane & 3, n = w.c1 - w.c0;
    const uint32_t sbase = smem_u32(sm);
    const int first = X == 1 ? self : self >> 1, x = X == 1 ? 0 : (self ^ lr) & 1;
    const uint32_t src = (first * 8 + lr) * D + q * 16 + x * 64, dst = (first * 8 + lr) * 128 + x * 16384;
    const uint32_t ca = dst + (((2 * q) ^ lr) << 4), cb = dst + (((2 * q + 1) ^ lr) << 4);
    int s = 0, round = 0;
    for (int p = 0; p < 2 * n; ++p, s = s + 1 == NS ? 0 : s + 1, round += s == 0) {
        const int o = p % NO;
        int c;
        bool value;
        tile_of(p, n, a.streams, &c, &value);
        if (!role_wait(&codes_full[s], round & 1, abort_flag, a.wait_ns)) break;
        if (p >= NO && !role_wait(&op_empty[o], (p / NO - 1) & 1, abort_flag, a.wait_ns)) break;
        const uint32_t from = sbase + Sh::codes_at(s) + src;
        const uint32_t to = sbase + Sh::kOffOps + o * Sh::kOperand;
        const uint32_t sc = sbase + Sh::kOffScales + ((w.c0 + c) % kChunks) * kGroups * 16;
        const int rows = __float_as_int(lds_f4(sc + (lane & 7) * 16).w);  // of 16 keys a lane
        const bool whole = __all_sync(0xFFFFFFFFu, rows == 16);
#pragma unroll
        for (int base = 0; base < STEPS; base += 4) {
            uint4 k[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (base + u < STEPS && (STEPS * BY == kChunk / 8 || first + (base + u) * BY < kChunk / 8))
                    k[u] = lds_u4(from + (base + u) * BY * 8 * D);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int step = first + (base + u) * BY;
                if (base + u >= STEPS || (STEPS * BY != kChunk / 8 && step >= kChunk / 8)) break;
                if (!whole && (step * 8 + lr & 15) >= __shfl_sync(0xFFFFFFFFu, rows, step >> 1)) k[u] = make_uint4(0, 0, 0, 0);
                const uint32_t line = to + (base + u) * BY * 1024;
                sts_u4(line + ca, halves_of<CODE>(k[u].x, 0), halves_of<CODE>(k[u].x, 1), halves_of<CODE>(k[u].y, 0),
                       halves_of<CODE>(k[u].y, 1));
                sts_u4(line + cb, halves_of<CODE>(k[u].z, 0), halves_of<CODE>(k[u].z, 1), halves_of<CODE>(k[u].w, 0),
                       halves_of<CODE>(k[u].w, 1));
            }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            mbar_arrive(&op_full[o]);
            mbar_arrive(&codes_empty[s]);
        }
    }
}

template <int CODE, int D>
__device__ __forceinline__ void convert(const QuantArgs& a, const Item& w, uint8_t* sm, uint64_t* codes_full,
                                        uint64_t* codes_empty, uint64_t* op_full, uint64_t* op_empty,
                                        volatile int* abort_flag, int self, int warps) {
    switch (warps) {  // a call has more than one warp of rows: fewer are the few-row kernel's
        case 2: return convert<CODE, D, 2>(a, w, sm, codes_full, codes_empty, op_full, op_empty, abort_flag, self);
        case 4: return convert<CODE, D, 4>(a, w, sm, codes_full, codes_empty, op_full, op_empty, abort_flag, self);
        default: return convert<CODE, D, 6>(a, w, sm, codes_full, codes_empty, op_full, op_empty, abort_flag, self);
    }
}

// GK: keys that share their scales (a page of 64 or 128 tokens: 64; else 16).
template <typename T, int CODE, int D, int GK>
__global__ void __launch_bounds__(kThreads, 1) quant_tile_kernel(const QuantArgs a) {
    using Sh = QuantTile<D>;
    constexpr int NO = Sh::kOps, KS = D / 16, kAll = Sh::kStages + Sh::kMore, FIRST = kFirst<D, GK>;
    extern __shared__ __align__(1024) uint8_t sm[];
    const int NS = a.streams ? kAll : Sh::kStages;
    const uint32_t sbase = smem_u32(sm);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Sh::kOffBar);
    uint64_t *codes_full = bars, *codes_empty = bars + kAll, *op_full = bars + 2 * kAll, *op_empty = op_full + NO,
             *bar_s = op_empty + NO, *bar_p = bar_s + 2, *bar_o = bar_p + 4, *bar_drain = bar_o + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + Sh::kOffMisc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + Sh::kOffMisc + 4);
    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    // Of one half's rows, the softmax warps without a row convert too.
    const int row_warps = a.streams ? (a.Tq * a.G + 31) / 32 : 4, converters = 2 + 2 * (4 - row_warps);
    if (warp == 1) tmem_alloc(tmem_slot, 512);
    if (threadIdx.x == 0) {
        for (int s = 0; s < kAll; ++s) {
            mbar_init(&codes_full[s], 2);   // the bytes, and the scales beside them
            mbar_init(&codes_empty[s], converters);
        }
        for (int s = 0; s < NO; ++s) {
            mbar_init(&op_full[s], converters);
            mbar_init(&op_empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar_s[i], 1);
            mbar_init(&bar_p[2 * i], row_warps);
            mbar_init(&bar_p[2 * i + 1], row_warps);
            mbar_init(&bar_o[i], 1);
        }
        mbar_init(bar_drain, 1);
        *abort_flag = a.wait_ns == 0;  // then the MMA thread gives up before its first wait, copies in flight
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    grid_wait();  // the inputs, the lengths among them, and the parts' last readers
    grid_trigger();
    const Item w = item_of(a);
    const int n = w.c1 - w.c0;
    Loader<D> loader;
    if (warp == 0) {  // the first tiles' copies are on their way while Q comes in
        __syncwarp();
        loader.start(a, w);
        for (int i = 0; i < NS && i < 2 * n; ++i) loader.load(a, w, sm, codes_full, i, i);
    } else {
        load_q<T, D>(a, w, sm);
    }
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp >= 4) {
        // 384 threads launch at 168 registers: 128 x 72 + 256 x 216 = 384 x 168
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;" ::: "memory");
        if ((warp & 3) < row_warps)
            softmax_half<T, D, GK>(a, w, sm, bar_s, bar_p, bar_o, abort_flag, tmem);
        else
            convert<CODE, D>(a, w, sm, codes_full, codes_empty, op_full, op_empty, abort_flag,
                             2 + (warp - 4 >> 2) * (4 - row_warps) + (warp & 3) - row_warps, converters);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;" ::: "memory");
        if (warp == 0) {
            int p = 2 * n < NS ? 2 * n : NS, s = 0, round = 0;
            for (; p < 2 * n; ++p) {
                if (!role_wait(&codes_empty[s], round & 1, abort_flag, a.wait_ns)) break;
                loader.load(a, w, sm, codes_full, p, s);
                if (++s == NS) s = 0, ++round;
            }
            // Every copy issued lands before the CTA leaves, also when it was another role that gave up.
            for (int i = p > NS ? p - NS : 0; i < p; ++i) mbar_wait_bounded(&codes_full[i % NS], (i / NS) & 1);
            __syncwarp();
        } else if (warp == 1) {
            // ------------------------------------------------ every MMA of the CTA, from one thread
            constexpr uint32_t idS = umma_idesc_f16<__half>(128, 128, false);
            constexpr uint32_t idO = umma_idesc_f16<__half>(128, D, true);
            if (elect_one()) {
                const uint64_t qd0 = sw128_desc(sbase, 16, 1024);
                const uint64_t kd0 = sw128_desc(sbase + Sh::kOffOps, 16, 1024);
                const uint64_t vd0 = sw128_desc(sbase + Sh::kOffOps, 16384, 1024);
                const uint32_t q1 = a.streams ? 0 : Sh::kOperand;
                int stage = 0, phase = 0;  // of the next tile of the ring
                auto advance = [&]() {
                    if (++stage == NO) stage = 0, phase ^= 1;
                };
                auto scores = [&](int hf, int st) {
                    const uint64_t qd = desc_at(qd0, hf ? q1 : 0), kd = desc_at(kd0, st * Sh::kOperand);
#pragma unroll
                    for (int kk = 0; kk < KS; ++kk) {
                        const uint32_t off = (kk >> 2) * 16384 + (kk & 3) * 32;
                        umma_f16_ss(tmem + hf * 128, desc_at(qd, off), desc_at(kd, off), idS, kk > 0);
                    }
                    umma_commit(&bar_s[hf]);
                };
                // P_h's first keys and the others as they come; O_h starts afresh on a half's first chunk
                auto product = [&](int hf, int st, bool fresh, uint32_t parity) -> bool {
                    const uint64_t vd = desc_at(vd0, st * Sh::kOperand);
                    const uint32_t o = tmem + 256 + hf * 128, p = tmem + hf * 128;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        if (!thread_wait(&bar_p[2 * hf + half], parity, abort_flag, a.wait_ns)) return false;
                        tc_fence_after();
#pragma unroll
                        for (int kk = FIRST * half; kk < (half ? kGroups : FIRST); ++kk)
                            umma_f16_ts(o, p + kk * 8, desc_at(vd, kk * 2048), idO, kk > 0 || !fresh);
                    }
                    return true;
                };
                auto tile = [&]() -> bool {
                    const bool ok = thread_wait(&op_full[stage], phase, abort_flag, a.wait_ns);
                    tc_fence_after();
                    return ok;
                };
                bool ok = *abort_flag == 0;
                if (ok && n > 0 && !a.streams) {
                    ok = tile();
                    if (ok) {
                        scores(0, stage), scores(1, stage);
                        umma_commit(&op_empty[stage]);
                        advance();
                    }
                    for (int j = 0; ok && j < n; ++j) {
                        const bool more = j + 1 < n;
                        const int sv = stage;
                        if (!(ok = tile())) break;
                        advance();
                        if (!(ok = product(0, sv, j == 0, j & 1))) break;
                        if (more) {
                            if (!(ok = tile())) break;
                            scores(0, stage);
                        }
                        if (!(ok = product(1, sv, j == 0, j & 1))) break;
                        umma_commit(&op_empty[sv]);
                        if (more) {
                            scores(1, stage);
                            umma_commit(&op_empty[stage]);
                            advance();
                        }
                    }
                } else if (ok && n > 0) {
                    for (int c = 0; ok && c < n && c < 2; ++c) {
                        ok = tile();
                        if (ok) {
                            scores(c, stage);
                            umma_commit(&op_empty[stage]);
                            advance();
                        }
                    }
                    for (int c = 0; ok && c < n; ++c) {
                        const int hf = c & 1;
                        if (!(ok = tile())) break;
                        if (!(ok = product(hf, stage, c < 2, (c >> 1) & 1))) break;
                        umma_commit(&op_empty[stage]);
                        advance();
                        if (c + 2 < n) {
                            if (!(ok = tile())) break;
                            scores(hf, stage);
                            umma_commit(&op_empty[stage]);
                            advance();
                        }
                    }
                }
                if (ok) umma_commit(&bar_o[0]), umma_commit(&bar_o[1]);
                umma_commit(bar_drain);  // every MMA completes before the TMEM is released
                mbar_wait_bounded(bar_drain, 0);
            }
            __syncwarp();
        } else {
            convert<CODE, D>(a, w, sm, codes_full, codes_empty, op_full, op_empty, abort_flag, warp - 2, converters);
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

template <typename T, int CODE, int D, int GK> int launch(const QuantArgs& a, unsigned grid, cudaStream_t stream) {
    if (!allow_kernel<quant_tile_kernel<T, CODE, D, GK>>(QuantTile<D>::kSmem)) return LSA_ERR_CUDA;
    return launch_after(quant_tile_kernel<T, CODE, D, GK>, dim3(grid), kThreads, QuantTile<D>::kSmem, stream, a);
}
template <typename T, int CODE, int D> int launch(const QuantArgs& a, unsigned grid, cudaStream_t stream) {
    return a.shift >= 6 ? launch<T, CODE, D, 64>(a, grid, stream) : launch<T, CODE, D, 16>(a, grid, stream);
}
template <typename T> int launch(const QuantArgs& a, int code, int D, unsigned grid, cudaStream_t stream) {
    if (code == kE4M3) return D == 128 ? launch<T, kE4M3, 128>(a, grid, stream) : launch<T, kE4M3, 64>(a, grid, stream);
    return D == 128 ? launch<T, kInt8, 128>(a, grid, stream) : launch<T, kInt8, 64>(a, grid, stream);
}

}  // namespace

int launch_quant_tiles(const QuantArgs& a, int dtype, int code, int D, cudaStream_t stream) {
    if (a.lists != nullptr || a.status == nullptr) return LSA_ERR_ARG;  // a read's: it has neither kernel nor status here
    if (a.streams && a.Tq * a.G <= 32) return LSA_ERR_ARG;  // convert() has no form for that many idle softmax warps
    const int64_t all = (int64_t)a.B * a.Hkv * a.tiles, items = a.whole + (all - a.whole) * a.parts;
    if (items > INT32_MAX) return LSA_ERR_SIZE;
    return dtype == kBF16 ? launch<__nv_bfloat16>(a, code, D, (unsigned)items, stream)
                          : launch<__half>(a, code, D, (unsigned)items, stream);
}

}  // namespace lsa
