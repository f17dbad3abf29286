// prefix_umma.cuh - what the tensor-core kernels of the shared-prefix attention share: bounded
// role waits, TMA tile loads, packed fp32 arithmetic, tensor maps (sm_100a).
#pragma once

#include <cuda.h>

#include "prefix.cuh"
#include "umma.cuh"

namespace lsa {

constexpr int kChunk = 128;  // keys of a tile

// Warp-uniform bounded wait on an mbarrier phase; false: it expired or another role gave up.
__device__ __forceinline__ bool role_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint64_t limit_ns) {
    bool done = mbar_try_wait(bar, parity);
    if (__all_sync(0xFFFFFFFFu, done)) return true;
    const uint64_t t0 = global_ns();
    for (;;) {
        if (!done) done = mbar_try_wait(bar, parity);
        if (__all_sync(0xFFFFFFFFu, done)) return true;
        int stop = 0;
        if ((threadIdx.x & 31) == 0) stop = (*abort_flag != 0) || (global_ns() - t0 > limit_ns);
        if (__shfl_sync(0xFFFFFFFFu, stop, 0)) {
            if ((threadIdx.x & 31) == 0) *abort_flag = 1;
            return false;
        }
    }
}

// The same for a role that is one thread; the flag and the clock are looked at now and then.
__device__ __forceinline__ bool thread_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint64_t limit_ns) {
    uint64_t t0 = 0;
    for (int i = 0;; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 15) == 15) {
            const uint64_t now = global_ns();
            if (t0 == 0) t0 = now;
            if (*abort_flag != 0 || now - t0 > limit_ns) {
                *abort_flag = 1;
                return false;
            }
        }
    }
}

// One lane of a converged warp. An MMA-issuing thread chosen this way issues a 128 x 128 x 16 MMA
// every 64 cycles, the pipe's rate, with barrier waits between them; chosen by lane == 0 it took
// 83-95 (measured on B200: the compiler knows the elected branch to be one thread).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred P;\n\t"
        "elect.sync _|P, 0xFFFFFFFF;\n\t"
        "selp.u32 %0, 1, 0, P;\n\t}"
        : "=r"(p));
    return p != 0;
}

// A 128-byte-swizzled operand's descriptor is base + (byte offset >> 4) in its low word: the
// start address stays within its 14 bits everywhere in shared memory.
__device__ __forceinline__ uint64_t desc_at(uint64_t base, uint32_t byte_offset) { return base + (byte_offset >> 4); }

__device__ __forceinline__ void tma_tile(uint32_t dst, const CUtensorMap* map, int x, int c1, int c2, int c3,
                                         uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
        "%5}], [%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
        : "memory");
}

// Untiled bulk copy shared -> global (16-byte aligned, whole multiples of 16 bytes), one group a
// thread: committed by the thread that issued it, which waits until shared memory has been read.
__device__ __forceinline__ void bulk_s2g(void* dst, uint32_t src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void bulk_commit_wait() {
    asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;" ::: "memory");
}

__device__ __forceinline__ uint32_t pack16(float a, float b, __nv_bfloat16*) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack16(float a, float b, __half*) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeFn encode_fn() {
    static EncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) !=
                cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

// tcgen05.st 32x32b.x16 (complete after tmem_wait_st).
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};"
        :
        : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// A 4-dimensional map of 16-bit elements (D innermost, then the three extents and strides given,
// in elements) with boxes of 64 x b1 x b2 x 1 elements, 128-byte swizzle, zeros past the extents.
inline bool encode_map(CUtensorMap* map, bool bf16, const void* base, int64_t D, int64_t n1, int64_t n2, int64_t n3,
                       int64_t s1, int64_t s2, int64_t s3, int b1, int b2) {
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)n1, (cuuint64_t)n2, (cuuint64_t)n3};
    const cuuint64_t strides[3] = {(cuuint64_t)s1 * 2, (cuuint64_t)s2 * 2, (cuuint64_t)s3 * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)b1, (cuuint32_t)b2, 1}, es[4] = {1, 1, 1, 1};
    return encode_fn()(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                       const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Keys [B, T, H, D]: boxes of 128 keys of one head.
inline bool encode_keys(CUtensorMap* map, bool bf16, const void* base, int64_t D, int64_t T, int64_t H, int64_t B,
                        int64_t st, int64_t sh, int64_t sb) {
    return encode_map(map, bf16, base, D, T, H, B, st, sh, sb, kChunk, 1);
}

}  // namespace lsa
