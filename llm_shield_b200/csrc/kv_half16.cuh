// What the paged-cache attention kernels share: the two 16-bit types, the
// exponential, and where a position's row lies.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "kv_launch.cuh"
#include "kv_ops.h"

namespace shield {
namespace kv {

template <bool BF16>
struct Half16;
template <>
struct Half16<false> {
    // f16 weights carry a factor (it cancels in o / sum), so that small ones are
    // still numbers and the largest is far from overflow: 2^14 in the few-row
    // kernel, where the row's largest weight is 1 (down to 2^-38 of it), 2^6 in the
    // many-row kernel, where the largest may have grown to 2^8 (down to 2^-30 of a
    // maximum just taken; below 2^-20 of it with fewer bits)
    static constexpr float LIFT = 14.0f;
    static constexpr uint32_t EXP = 0x7C00u;  // exponent bits: all ones in infinities and NaN
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 r = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&r);
    }
    static __device__ __forceinline__ float value(uint16_t x) { return __half2float(__ushort_as_half(x)); }
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <>
struct Half16<true> {
    static constexpr float LIFT = 0.0f;
    static constexpr uint32_t EXP = 0x7F80u;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&r);
    }
    static __device__ __forceinline__ float value(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

// Two packed values: bits 15 and 31 tell which of them is not finite (adding the
// exponent's lowest bit carries out of it only where it is all ones).
template <bool BF16>
__device__ __forceinline__ uint32_t not_finite_bits(uint32_t w) {
    constexpr uint32_t E = Half16<BF16>::EXP, E2 = E | E << 16, ONE = (E & (~E + 1)) * 0x10001u;
    return ((w & E2) + ONE) & 0x80008000u;
}
// The pair with such values as 0.
template <bool BF16>
__device__ __forceinline__ uint32_t finite_part(uint32_t w) {
    constexpr uint32_t E = Half16<BF16>::EXP;
    if ((w & E) == E) w &= 0xFFFF0000u;
    if (((w >> 16) & E) == E) w &= 0x0000FFFFu;
    return w;
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Lets a kernel use `bytes` of shared memory, once per device (`done`: a bit for
// each of the first 64; calls from several host threads set the same).
template <class K>
inline cudaError_t allow_smem(K kernel, int bytes, std::atomic<uint64_t> &done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// First element of position `row` of a page: layer, page, kv head.
__device__ __forceinline__ int64_t row_offset(const DevPool &P, int layer, int page, int head, int row) {
    return (int64_t)layer * P.layer_stride() +
           ((((int64_t)page * P.kv_heads + head) << P.page_shift) + row) * P.dim;
}

}  // namespace kv
}  // namespace shield
