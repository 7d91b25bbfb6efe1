// Paged-cache kernels that move rows: pages to pages (fork, copy, compact) and
// a step's new keys and values to their slots. Both only move bytes; their
// bound is HBM bandwidth, or launch latency for a few rows: 24 sequences of
// 200-1000 tokens copied and packed 6.6 TB/s (the measured copy rate), 256 forks'
// partial pages 6.6 TB/s in the kernel, 16,384 rows of 2 x 1024 bf16 5.4 TB/s.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstring>

#include "kv_launch.cuh"
#include "kv_ops.h"

namespace shield {
namespace kv {

// The list of moves travels in the launch's parameters, so no staging buffer
// has to outlive the call; longer lists take several launches.
template <int N>
struct MoveList {
    Move m[N];
};

// One CTA per (move, layer, keys or values): the page's rows lie head by head,
// page_tokens * dim elements apart, and are copied in 16-byte vectors.
template <int N>
__global__ void __launch_bounds__(256) k_move_pages(const __grid_constant__ MoveList<N> list, const DevPool pool) {
    const Move mv = list.m[blockIdx.x];
    const int layer = blockIdx.y >> 1;
    char *base = static_cast<char *>(blockIdx.y & 1 ? pool.v : pool.k);
    const int64_t head_bytes = (int64_t)pool.page_tokens * pool.dim * 2;
    const int64_t page_bytes = head_bytes * pool.kv_heads;
    base += (int64_t)layer * pool.pages * page_bytes;
    const char *src = base + mv.src * page_bytes;
    char *dst = base + mv.dst * page_bytes;
    const int vecs = mv.rows * pool.dim / 8;  // 16-byte vectors of one head's rows
    const int total = vecs * pool.kv_heads;
    // eight vectors of a thread are on their way together
    for (int i0 = threadIdx.x; i0 < total; i0 += 8 * 256) {
        uint4 x[8];
        int64_t off[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int i = i0 + j * 256;
            if (i >= total) break;
            off[j] = (int64_t)(i / vecs) * head_bytes + (int64_t)(i % vecs) * 16;
            x[j] = *reinterpret_cast<const uint4 *>(src + off[j]);
        }
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (i0 + j * 256 < total) *reinterpret_cast<uint4 *>(dst + off[j]) = x[j];
    }
}

template <int N>
static cudaError_t move_some(const DevPool &pool, const Move *moves, int n, cudaStream_t s) {
    MoveList<N> list;
    memcpy(list.m, moves, (size_t)n * sizeof(Move));
    return launch(k_move_pages<N>, dim3((unsigned)n, (unsigned)pool.layers * 2), 256, 0, false, s, list, pool);
}

cudaError_t launch_move_pages(const DevPool &pool, const Move *moves, int64_t n, cudaStream_t s) {
    for (int64_t i = 0; i < n;) {
        const int64_t left = n - i;
        const int take = (int)std::min<int64_t>(left, 300);
        const cudaError_t e = take <= 32 ? move_some<32>(pool, moves + i, take, s) : move_some<300>(pool, moves + i, take, s);
        if (e != cudaSuccess) return e;
        i += take;
    }
    return cudaSuccess;
}

__device__ __forceinline__ uint32_t pack_pair(float a, float b, bool bf16) {
    if (bf16) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&r);
    }
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&r);
}

// A thread moves 8 values of a row at a time (one 16-byte store); f32 sources are
// rounded once, to nearest even. blockIdx.y: 0 keys, 1 values.
template <bool F32>
__global__ void __launch_bounds__(256) k_write_rows(const DevPool pool, const DevPlan plan, int layer, const void *k,
                                                    int64_t k_stride, const void *v, int64_t v_stride) {
    const int per_tok = pool.kv_heads * pool.dim / 8;
    const int64_t n = (int64_t)plan.counts[COUNT_TOKENS] * per_tok;
    const char *src = static_cast<const char *>(blockIdx.y ? v : k);
    const int64_t stride = blockIdx.y ? v_stride : k_stride;
    uint16_t *dst = static_cast<uint16_t *>(blockIdx.y ? pool.v : pool.k) + (int64_t)layer * pool.layer_stride();
    const int per_head = pool.dim / 8;
    // four vectors of a thread are on their way together
    constexpr int AT_ONCE = 4;
    for (int64_t i0 = (int64_t)blockIdx.x * (256 * AT_ONCE) + threadIdx.x; i0 < n; i0 += (int64_t)gridDim.x * (256 * AT_ONCE)) {
        uint4 o[AT_ONCE];
        int64_t to[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; j++) {
            const int64_t i = i0 + j * 256;
            if (i >= n) break;
            const int64_t t = i / per_tok;
            const int c = (int)(i - t * per_tok), h = c / per_head, d = (c - h * per_head) * 8;
            const int slot = plan.slot[t];
            const int64_t page = slot >> pool.page_shift, row = slot & (pool.page_tokens - 1);
            to[j] = (((page * pool.kv_heads + h) << pool.page_shift) + row) * pool.dim + d;
            if (F32) {
                const float4 *p = reinterpret_cast<const float4 *>(src + (t * stride + c * 8) * 4);
                const float4 a = p[0], b = p[1];
                o[j] = make_uint4(pack_pair(a.x, a.y, pool.bf16), pack_pair(a.z, a.w, pool.bf16),
                                  pack_pair(b.x, b.y, pool.bf16), pack_pair(b.z, b.w, pool.bf16));
            } else {
                o[j] = *reinterpret_cast<const uint4 *>(src + (t * stride + c * 8) * 2);
            }
        }
#pragma unroll
        for (int j = 0; j < AT_ONCE; j++)
            if (i0 + j * 256 < n) *reinterpret_cast<uint4 *>(dst + to[j]) = o[j];
    }
}

// Four values a thread.
__global__ void __launch_bounds__(256) k_narrow(const float4 *__restrict__ x, uint2 *__restrict__ y, int64_t n4, bool bf16) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n4) return;
    const float4 v = x[i];
    y[i] = make_uint2(pack_pair(v.x, v.y, bf16), pack_pair(v.z, v.w, bf16));
}
__global__ void __launch_bounds__(256) k_widen(const uint2 *__restrict__ x, float4 *__restrict__ y, int64_t n4, bool bf16) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n4) return;
    const uint2 v = x[i];
    if (bf16) {
        y[i] = make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xFFFF0000u), __uint_as_float(v.y << 16),
                           __uint_as_float(v.y & 0xFFFF0000u));
    } else {
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&v.y));
        y[i] = make_float4(a.x, a.y, b.x, b.y);
    }
}

cudaError_t launch_narrow(const float *x, void *y, int64_t n, bool bf16, cudaStream_t s) {
    if (n % 4) return cudaErrorInvalidValue;
    if (n == 0) return cudaSuccess;
    return launch(k_narrow, (unsigned)((n / 4 + 255) / 256), 256, 0, false, s, reinterpret_cast<const float4 *>(x), static_cast<uint2 *>(y),
                  n / 4, bf16);
}

cudaError_t launch_widen(const void *x, float *y, int64_t n, bool bf16, cudaStream_t s) {
    if (n % 4) return cudaErrorInvalidValue;
    if (n == 0) return cudaSuccess;
    return launch(k_widen, (unsigned)((n / 4 + 255) / 256), 256, 0, false, s, static_cast<const uint2 *>(x), reinterpret_cast<float4 *>(y),
                  n / 4, bf16);
}

cudaError_t launch_write_rows(const DevPool &pool, const DevPlan &plan, int64_t tokens, int32_t layer, bool f32,
                              const void *k, int64_t k_stride, const void *v, int64_t v_stride, cudaStream_t s) {
    const int64_t n = tokens * pool.kv_heads * pool.dim / 8;
    if (n == 0) return cudaSuccess;
    const dim3 grid((unsigned)std::min<int64_t>((n + 1023) / 1024, 1 << 20), 2);
    return launch(f32 ? k_write_rows<true> : k_write_rows<false>, grid, 256, 0, false, s, pool, plan, layer, k, k_stride, v, v_stride);
}

}  // namespace kv
}  // namespace shield
