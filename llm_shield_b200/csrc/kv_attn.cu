// Attention of a batch of sequences over a paged cache.
//
// For a token at position p and query head h of the group of kv head j:
//   o = sum_{l <= p} w_l v_l / sum w_l,   w_l = 2^(s_l - m),  s_l = scale log2(e) q.k_l
// with m the running maximum of s. The plan (kv_pool.h) cuts the keys into
// segments: runs of pages that several sequences share, computed once for the
// rows of all of them, and the rest of each sequence. A row whose keys lie in
// several pieces gets a partial (m, sum, unnormalised o) from each, joined by
// k_attend_merge. Scores, maxima, sums and outputs are f32; the weights are
// rounded to the cache's type for the product with the values (one rounding of
// at most half a step, as the output itself has).
#include <algorithm>

#include "kv_half16.cuh"
#include "kv_ops.h"

namespace shield {
namespace kv {

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}

// ------------------------------------------------------------- few rows

// Up to 16 rows (a decode step's group of query heads, a short draft) against
// a run of keys: bound by reading the keys and values once. Four warps take
// every fourth tile of 16 keys each, with a running (m, sum, o) of their own
// and their own ring of cp.async stages, so no warp waits for another until
// the four are joined at the end. Where the plan has more short pieces (up to
// FEW_SOLO keys) than the GPU holds CTAs, a warp takes one alone: such a piece
// is a chain of lookups and loads whose latency, not whose work, fills its
// time, and four times as many are on their way (with the kernels' early
// launches, a step of 128 sequences with 1-256 keys of their own: 63 -> 50 us).
template <int D>
struct FewShape {
    static constexpr int WARPS = 4;
    static constexpr int KEYS = 16;  // keys of a tile; pages hold a multiple
    static constexpr int STAGES = D == 128 ? 3 : 4;
    static constexpr int TILE_BYTES = KEYS * D * 2;
    static constexpr int STAGE_BYTES = 2 * TILE_BYTES;  // keys, values
    static constexpr int RING_BYTES = WARPS * STAGES * STAGE_BYTES;
    static constexpr int JOIN_LD = D + 8;  // floats from row to row of a warp's output: no bank conflicts
    static constexpr int JOIN_BYTES = WARPS * 16 * JOIN_LD * 4;
    static_assert(16 * JOIN_LD * 4 <= STAGES * STAGE_BYTES, "a lone warp's output takes its ring's place");
    static constexpr int BYTES = RING_BYTES > JOIN_BYTES ? RING_BYTES : JOIN_BYTES;
};

template <bool BF16, int D>
__global__ void __launch_bounds__(128, 2) k_attend_few(const AttendArgs A) {
    using S = FewShape<D>;
    using H = Half16<BF16>;
    extern __shared__ __align__(128) uint8_t few_smem[];
    __shared__ float2 join_ml[S::WARPS][16];
    __shared__ int dirty;
    const DevPool &P = A.pool;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.launch_dependents;");
    const int alone = (A.solo >= 0 ? A.solo : A.plan.counts[COUNT_SOLO]) * P.kv_heads;  // the last units of the list
    const int shared = (A.few >= 0 ? A.few : A.plan.counts[COUNT_FEW]) * P.kv_heads - alone;
    uint8_t *const own_smem = few_smem + warp * S::STAGES * S::STAGE_BYTES;
    const uint32_t ring = smem_addr(own_smem);
    for (int task = blockIdx.x; task < shared + (alone + S::WARPS - 1) / S::WARPS; task += gridDim.x) {
        const bool solo = task >= shared;
        const int u = solo ? shared + (task - shared) * S::WARPS + warp : task;
        if (solo && u >= shared + alone) continue;  // nothing below is waited for by other warps
        const int first = solo ? 0 : warp, step = solo ? 1 : S::WARPS;  // this warp's tiles
        const Item it = A.plan.few[u / P.kv_heads];
        const int kvh = u % P.kv_heads;
        const int32_t *table = A.plan.table + it.table;
        const int ntiles = (it.k1 - it.k0 + S::KEYS - 1) / S::KEYS;
        if (threadIdx.x == 0 && !solo) dirty = 0;

        // The page list in registers, a page per lane, 32 pages and the next 32, so
        // that no load waits for its page number.
        const int32_t *const list = table + (it.k0 >> P.page_shift);
        const int npages = (it.k1 - it.k0 + P.page_tokens - 1) >> P.page_shift;
        int window = 0;
        int here = lane < npages ? list[lane] : 0, next = 32 + lane < npages ? list[32 + lane] : 0;
        auto load = [&](int t, int stage) {
            const int p0 = it.k0 + t * S::KEYS;
            int pg = (t * S::KEYS >> P.page_shift) - window;
            if (pg >= 32) {  // (a warp's tiles are less than 32 pages apart)
                pg -= 32;
                window += 32;
                here = next;
                next = window + 32 + lane < npages ? list[window + 32 + lane] : 0;
            }
            const int64_t off = row_offset(P, A.layer, __shfl_sync(0xffffffffu, here, pg), kvh, p0 & (P.page_tokens - 1));
            const uint16_t *k = static_cast<const uint16_t *>(P.k) + off, *v = static_cast<const uint16_t *>(P.v) + off;
            const uint32_t dst = ring + stage * S::STAGE_BYTES;
#pragma unroll
            for (int i = 0; i < S::KEYS * D / 8 / 32; i++) {
                const int idx = i * 32 + lane, row = idx / (D / 8), c = idx % (D / 8);
                const bool ok = p0 + row < it.k1;
                const uint32_t to = row * D * 2 + ((c ^ (row & 7)) << 4);
                copy16(dst + to, ok ? k + idx * 8 : k, ok);
                copy16(dst + S::TILE_BYTES + to, ok ? v + idx * 8 : v, ok);
            }
        };
#pragma unroll
        for (int s = 0; s < S::STAGES - 1; s++) {
            if (first + s * step < ntiles) load(first + s * step, s);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }

        // this thread's rows: lane / 4 and lane / 4 + 8
        uint32_t qf[D / 16][4];
        int lim[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = (lane >> 2) + 8 * e;
            lim[e] = it.k1;
            const uint16_t *q = nullptr;
            if (r < it.nr) {
                const int at = it.tok0 + (it.r0 + r) / A.group, head = kvh * A.group + (it.r0 + r) % A.group;
                lim[e] = A.plan.lim[at];
                q = static_cast<const uint16_t *>(A.q) + A.plan.perm[at] * A.q_stride + head * D + (lane & 3) * 2;
            }
#pragma unroll
            for (int kk = 0; kk < D / 16; kk++) {
                qf[kk][e] = q ? *reinterpret_cast<const uint32_t *>(q + kk * 16) : 0;
                qf[kk][2 + e] = q ? *reinterpret_cast<const uint32_t *>(q + kk * 16 + 8) : 0;
            }
        }
        // the token whose row this thread helps to write at the end
        const int mine = solo ? min(lane, it.nr - 1) : min((int)threadIdx.x >> 3, it.nr - 1);
        const int token = A.plan.perm[it.tok0 + (it.r0 + mine) / A.group];
        const int low = it.masked ? A.plan.lim[it.tok0 + it.r0 / A.group] : it.k1;  // below it every row sees every key

        float m[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
        float o[D / 8][4];
#pragma unroll
        for (int i = 0; i < D / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        bool found = false;

        int stage = 0;
        for (int t = first; t < ntiles; t += step) {
            asm volatile("cp.async.wait_group %0;" ::"n"(S::STAGES - 2) : "memory");
            __syncwarp();
            const uint32_t ks = ring + stage * S::STAGE_BYTES, vs = ks + S::TILE_BYTES;
            const int p0 = it.k0 + t * S::KEYS;
            // two chains of products per 8 keys, even and odd steps of 16 dims
            float c[2][4], c1[2][4];
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) c[j][i] = c1[j][i] = 0.0f;
            const int mi = lane >> 3, mr = lane & 7;
#pragma unroll
            for (int kk = 0; kk < D / 16; kk++) {
                uint32_t b[4];
                ldsm4(b, ks + ((mi >> 1) * 8 + mr) * D * 2 + (((2 * kk + (mi & 1)) ^ mr) << 4));
                H::mma(kk & 1 ? c1[0] : c[0], qf[kk], b[0], b[1]);
                H::mma(kk & 1 ? c1[1] : c[1], qf[kk], b[2], b[3]);
            }
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) c[j][i] += c1[j][i];
            const bool masked = p0 + S::KEYS > low;
            if (masked) {
                // values that a row may not see must not reach its product as 0 * inf:
                // they count as 0 here, and rows that do see them get them at the end
#pragma unroll
                for (int i = 0; i < S::KEYS * D / 8 / 32; i++) {
                    const uint32_t a = vs + (i * 32 + lane) * 16;
                    uint32_t w[4];
                    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a) : "memory");
                    if (not_finite_bits<BF16>(w[0]) | not_finite_bits<BF16>(w[1]) | not_finite_bits<BF16>(w[2]) | not_finite_bits<BF16>(w[3])) {
                        found = true;
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(finite_part<BF16>(w[0])),
                                     "r"(finite_part<BF16>(w[1])), "r"(finite_part<BF16>(w[2])),
                                     "r"(finite_part<BF16>(w[3])) : "memory");
                    }
                }
                __syncwarp();
            }
            uint32_t pf[4];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float s[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    s[j] = c[j >> 1][2 * e + (j & 1)] * A.scale_log2;
                    if (masked && p0 + (j >> 1) * 8 + (lane & 3) * 2 + (j & 1) >= lim[e]) s[j] = -INFINITY;
                }
                float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = fmaxf(m[e], mx);
                const float ref = mn == -INFINITY ? 0.0f : mn;  // a row with no key so far keeps weights of 0
                const float old = exp2_approx(m[e] - ref), lift = ref - H::LIFT;
                m[e] = mn;
                float p[4];
#pragma unroll
                for (int j = 0; j < 4; j++) p[j] = exp2_approx(s[j] - lift);
                sum[e] = __fmaf_rn(sum[e], old, (p[0] + p[1]) + (p[2] + p[3]));
#pragma unroll
                for (int i = 0; i < D / 8; i++) {
                    o[i][2 * e] *= old;
                    o[i][2 * e + 1] *= old;
                }
                pf[e] = H::pack(p[0], p[1]);
                pf[2 + e] = H::pack(p[2], p[3]);
            }
#pragma unroll
            for (int np = 0; np < D / 16; np++) {
                uint32_t b[4];
                ldsm4_trans(b, vs + ((mi & 1) * 8 + mr) * D * 2 + (((2 * np + (mi >> 1)) ^ mr) << 4));
                H::mma(o[2 * np], pf, b[0], b[1]);
                H::mma(o[2 * np + 1], pf, b[2], b[3]);
            }
            __syncwarp();
            const int ahead = t + (S::STAGES - 1) * step;
            if (ahead < ntiles) load(ahead, stage == 0 ? S::STAGES - 1 : stage - 1);
            asm volatile("cp.async.commit_group;" ::: "memory");
            stage = stage + 1 == S::STAGES ? 0 : stage + 1;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
        for (int e = 0; e < 2; e++) {
            sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 1);
            sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 2);
        }
        // Writes four dims of a row, which the warps' outputs add up to.
        auto put = [&](int r, int tok, int d, float4 x, float M, float L, bool fix) {
            if (fix) {
                const int end = min(it.k1, A.plan.lim[it.tok0 + (it.r0 + r) / A.group]);
                for (int p = it.k0 + (max(low - it.k0, 0) / S::KEYS) * S::KEYS; p < end; p++) {
                    const uint16_t *v = static_cast<const uint16_t *>(P.v) +
                        row_offset(P, A.layer, table[p >> P.page_shift], kvh, p & (P.page_tokens - 1)) + d;
                    if ((v[0] & H::EXP) == H::EXP) x.x += H::value(v[0]);
                    if ((v[1] & H::EXP) == H::EXP) x.y += H::value(v[1]);
                    if ((v[2] & H::EXP) == H::EXP) x.z += H::value(v[2]);
                    if ((v[3] & H::EXP) == H::EXP) x.w += H::value(v[3]);
                }
            }
            if (it.part < 0) {
                const float inv = 1.0f / L;
                const int head = kvh * A.group + (it.r0 + r) % A.group;
                uint16_t *out = static_cast<uint16_t *>(A.out) + tok * A.out_stride + head * D + d;
                *reinterpret_cast<uint2 *>(out) = make_uint2(H::pack(x.x * inv, x.y * inv), H::pack(x.z * inv, x.w * inv));
            } else {
                const int64_t part = it.part + (int64_t)kvh * it.nr + r;
                *reinterpret_cast<float4 *>(A.plan.part_o + part * D + d) = x;
                if (d == 0) A.plan.part_ml[part] = make_float2(M, L);
            }
        };
        if (solo) {
            const bool fix = __any_sync(0xffffffffu, found);
            float *join = reinterpret_cast<float *>(own_smem);  // this warp's ring is free
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int r = (lane >> 2) + 8 * e;
                if ((lane & 3) == 0) join_ml[warp][r] = make_float2(m[e], sum[e]);
#pragma unroll
                for (int i = 0; i < D / 8; i++)
                    *reinterpret_cast<float2 *>(join + r * S::JOIN_LD + i * 8 + (lane & 3) * 2) = make_float2(o[i][2 * e], o[i][2 * e + 1]);
            }
            __syncwarp();
            for (int i0 = 0; i0 < it.nr * (D / 4); i0 += 32) {
                const int i = i0 + lane, r = i / (D / 4), d = i % (D / 4) * 4;
                const int tok = __shfl_sync(0xffffffffu, token, r & 15);
                if (r >= it.nr) continue;
                const float2 ml = join_ml[warp][r];
                put(r, tok, d, *reinterpret_cast<const float4 *>(join + r * S::JOIN_LD + d), ml.x, ml.y, fix);
            }
            __syncwarp();  // the ring is free for the next unit
            continue;
        }
        __syncthreads();  // every warp is done with its ring; dirty is set to 0
        float *join = reinterpret_cast<float *>(few_smem);
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = (lane >> 2) + 8 * e;
            if ((lane & 3) == 0) join_ml[warp][r] = make_float2(m[e], sum[e]);
#pragma unroll
            for (int i = 0; i < D / 8; i++)
                *reinterpret_cast<float2 *>(join + (warp * 16 + r) * S::JOIN_LD + i * 8 + (lane & 3) * 2) =
                    make_float2(o[i][2 * e], o[i][2 * e + 1]);
        }
        if (found) dirty = 1;
        __syncthreads();
        // 8 threads per row, each D / 8 dims in groups of 4
        const int r = threadIdx.x >> 3;
        if (r < it.nr) {
            float M = -INFINITY, L = 0.0f, w[S::WARPS];
#pragma unroll
            for (int i = 0; i < S::WARPS; i++) M = fmaxf(M, join_ml[i][r].x);
#pragma unroll
            for (int i = 0; i < S::WARPS; i++) {
                w[i] = exp2_approx(join_ml[i][r].x - (M == -INFINITY ? 0.0f : M));
                L = __fmaf_rn(join_ml[i][r].y, w[i], L);
            }
#pragma unroll
            for (int j = 0; j < D / 32; j++) {
                const int d = j * 32 + (threadIdx.x & 7) * 4;
                float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int i = 0; i < S::WARPS; i++) {
                    const float4 x = *reinterpret_cast<const float4 *>(join + (i * 16 + r) * S::JOIN_LD + d);
                    a.x = __fmaf_rn(x.x, w[i], a.x);
                    a.y = __fmaf_rn(x.y, w[i], a.y);
                    a.z = __fmaf_rn(x.z, w[i], a.z);
                    a.w = __fmaf_rn(x.w, w[i], a.w);
                }
                put(r, token, d, a, M, L, dirty != 0);
            }
        }
        __syncthreads();  // the ring and join_ml are free for the next unit
    }
    // (launched while the many-row kernel still runs: this one is not over before that is)
    if (blockIdx.x == gridDim.x - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <bool BF16, int D>
static cudaError_t few_launch(const AttendArgs &A, int64_t units, bool beside, cudaStream_t s) {
    using S = FewShape<D>;
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t e = allow_smem(k_attend_few<BF16, D>, S::BYTES, allowed);
    if (e != cudaSuccess) return e;
    return launch(k_attend_few<BF16, D>, (unsigned)units, 128, S::BYTES, beside, s, A);
}

cudaError_t launch_attend_few(const AttendArgs &A, int64_t units, bool beside, cudaStream_t s) {
    if (units == 0) return cudaSuccess;
    if (A.pool.dim == 128) return A.pool.bf16 ? few_launch<true, 128>(A, units, beside, s) : few_launch<false, 128>(A, units, beside, s);
    if (A.pool.dim == 64) return A.pool.bf16 ? few_launch<true, 64>(A, units, beside, s) : few_launch<false, 64>(A, units, beside, s);
    return cudaErrorInvalidValue;
}

// ----------------------------------------------------------------- joining

// One warp per (token, query head): 11 partials of 4096 rows of 128 in 6.7 us.
// The row's partials lie one per piece of keys of each segment on the way from
// the sequence's own keys up through the runs it shares, always in that order.
// A lane looks up one piece, so that the lookups of up to 32 pieces and the
// reads of their outputs go out together. (Dim 64: 32 registers, 12 bytes
// spilled.)
template <bool BF16, int D>
__global__ void __launch_bounds__(128) k_attend_merge(const AttendArgs A) {
    using H = Half16<BF16>;
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const int heads = A.group * A.pool.kv_heads;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // launched early: the partials are there from here on
    const int64_t rows = (int64_t)A.plan.counts[COUNT_MERGE] * heads;
    for (int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5); w < rows; w += (int64_t)gridDim.x * 4) {
        const Join J = A.plan.merge[w / heads];
        const int head = (int)(w % heads), kvh = head / A.group;
        float M = -INFINITY, L = 0.0f, o[E];
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = 0.0f;
        for (int sg = J.leaf; sg >= 0;) {
            const Segment S = A.plan.segs[sg];
            const int r = (J.at - S.tok0) * A.group + head % A.group, tile = r / S.tile_rows, in_tile = r % S.tile_rows;
            const int nr = min(S.tile_rows, S.rows - tile * S.tile_rows);
            for (int s0 = 0; s0 < S.nsplit; s0 += 32) {
                const int n = min(32, S.nsplit - s0);
                int part = lane < n ? A.plan.where[S.slot0 + (s0 + lane) * S.ntiles + tile] : -1;
                float2 ml = make_float2(-INFINITY, 0.0f);
                if (part >= 0) {
                    part += kvh * nr + in_tile;
                    ml = A.plan.part_ml[part];
                }
                float top = ml.x;
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float mn = fmaxf(M, top), ref = mn == -INFINITY ? 0.0f : mn;
                const float old = exp2_approx(M - ref), f = exp2_approx(ml.x - ref);
                M = mn;
                float l = ml.y * f;
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
                L = __fmaf_rn(L, old, l);
#pragma unroll
                for (int e = 0; e < E; e++) o[e] *= old;
#pragma unroll 8
                for (int s = 0; s < n; s++) {
                    const int p = __shfl_sync(0xffffffffu, part, s);
                    const float g = __shfl_sync(0xffffffffu, f, s);
                    if (p < 0) continue;
                    const float *src = A.plan.part_o + (int64_t)p * D + lane * E;
                    if constexpr (E == 4) {
                        const float4 x = *reinterpret_cast<const float4 *>(src);
                        o[0] = __fmaf_rn(x.x, g, o[0]);
                        o[1] = __fmaf_rn(x.y, g, o[1]);
                        o[2] = __fmaf_rn(x.z, g, o[2]);
                        o[3] = __fmaf_rn(x.w, g, o[3]);
                    } else {
                        const float2 x = *reinterpret_cast<const float2 *>(src);
                        o[0] = __fmaf_rn(x.x, g, o[0]);
                        o[1] = __fmaf_rn(x.y, g, o[1]);
                    }
                }
            }
            sg = S.parent;
        }
        const float inv = 1.0f / L;
        uint16_t *out = static_cast<uint16_t *>(A.out) + J.token * A.out_stride + head * D + lane * E;
        if constexpr (E == 4) *reinterpret_cast<uint2 *>(out) = make_uint2(H::pack(o[0] * inv, o[1] * inv), H::pack(o[2] * inv, o[3] * inv));
        else *reinterpret_cast<uint32_t *>(out) = H::pack(o[0] * inv, o[1] * inv);
    }
}

template <bool BF16, int D>
static cudaError_t merge_launch(const AttendArgs &A, int64_t tokens, cudaStream_t s) {
    const int64_t rows = tokens * A.group * A.pool.kv_heads;
    return launch(k_attend_merge<BF16, D>, (unsigned)std::min<int64_t>((rows + 3) / 4, 1 << 30), 128, 0, true, s, A);
}

cudaError_t launch_attend_merge(const AttendArgs &A, int64_t tokens, cudaStream_t s) {
    if (tokens == 0) return cudaSuccess;
    if (A.pool.dim == 128) return A.pool.bf16 ? merge_launch<true, 128>(A, tokens, s) : merge_launch<false, 128>(A, tokens, s);
    if (A.pool.dim == 64) return A.pool.bf16 ? merge_launch<true, 64>(A, tokens, s) : merge_launch<false, 64>(A, tokens, s);
    return cudaErrorInvalidValue;
}

}  // namespace kv
}  // namespace shield
