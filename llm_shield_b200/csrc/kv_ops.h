// Host-side launchers of the paged-cache kernels (kv_ops.cu, kv_attn.cu).
// Every launcher is asynchronous on the given stream and allocates nothing.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kv_pool.h"

namespace shield {
namespace kv {

// A pool on the device: K and V as [layers][pages][kv heads][page tokens][dims]
// of 16-bit floats (bf16 or f16).
struct DevPool {
    void *k = nullptr, *v = nullptr;
    bool bf16 = false;
    int32_t layers = 0, pages = 0, kv_heads = 0, page_tokens = 0, page_shift = 0, dim = 0;
    constexpr int64_t layer_stride() const { return (int64_t)pages * kv_heads * page_tokens * dim; }
};

// A batch's plan in device memory. Every array has a fixed place sized for the
// batch's capacities and the counts live beside them, so a captured launch
// reads whatever plan was uploaded last.
struct DevPlan {
    const int32_t *counts = nullptr;  // tokens, few items, tile items, tokens to join, few items for a warp alone
    const int32_t *slot = nullptr, *perm = nullptr, *lim = nullptr, *where = nullptr, *table = nullptr;
    const Join *merge = nullptr;
    const Segment *segs = nullptr;
    const Item *few = nullptr, *tile = nullptr;
    float *part_o = nullptr;   // [partial row][dim], not divided by the row's sum
    float2 *part_ml = nullptr; // running maximum (base-2 exponent) and sum of each partial row
};
enum { COUNT_TOKENS = 0, COUNT_FEW = 1, COUNT_TILE = 2, COUNT_MERGE = 3, COUNT_SOLO = 4, COUNTS = 5 };

struct AttendArgs {
    DevPool pool;
    DevPlan plan;
    const void *q = nullptr;
    void *out = nullptr;
    int64_t q_stride = 0, out_stride = 0;  // elements from token to token
    int32_t layer = 0, group = 1;
    int32_t few = -1, solo = -1, tile = -1;  // the plan's counts where the host knows them: one lookup less
    float scale_log2 = 0.0f;               // scale * log2(e)
    int32_t *err = nullptr;                // error word of bounded waits
};

// rows moves.rows of each page, every layer and head, keys and values.
cudaError_t launch_move_pages(const DevPool &pool, const Move *moves, int64_t n, cudaStream_t s);
// Tokens' keys and values (rows of kv_heads * dim, `stride` elements apart; f32
// or the pool's type) to their slots of one layer. tokens: the plan's, or an
// upper bound of later plans' (the kernel stops at the plan's count).
cudaError_t launch_write_rows(const DevPool &pool, const DevPlan &plan, int64_t tokens, int32_t layer, bool f32,
                              const void *k, int64_t k_stride, const void *v, int64_t v_stride, cudaStream_t s);
// n f32 values rounded to the pool's type, and 16-bit values widened to f32.
cudaError_t launch_narrow(const float *x, void *y, int64_t n, bool bf16, cudaStream_t s);
cudaError_t launch_widen(const void *x, float *y, int64_t n, bool bf16, cudaStream_t s);
// The three attention kernels over `units` work units (or CTAs for as many as a
// later plan may have: each strides over the plan's own count).
// beside: launch_attend_tile came just before, and this one may run beside it.
cudaError_t launch_attend_few(const AttendArgs &A, int64_t units, bool beside, cudaStream_t s);
// maps: map_pool of the keys and of the values, made once per pool.
bool map_pool(CUtensorMap *m, const DevPool &pool, void *data);
cudaError_t launch_attend_tile(const AttendArgs &A, const CUtensorMap *maps, int64_t units, int sms, cudaStream_t s);  // one persistent CTA per SM
cudaError_t launch_attend_merge(const AttendArgs &A, int64_t tokens, cudaStream_t s);

}  // namespace kv
}  // namespace shield
