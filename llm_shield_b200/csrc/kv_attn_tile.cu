// Attention of many rows over a paged cache, on the 5th-generation tensor
// cores: prompts, and runs of keys that a whole batch shares.
//
// A work unit is an item of the plan (up to 256 rows: tokens times the query
// heads of one kv head) and its run of keys, taken in blocks of 128. Per row
// tile of 128 rows and key block:
//   S = Q K^T   tcgen05.mma, both operands in shared memory, S in TMEM
//   P = 2^(scale S - m), rounded to the cache's type, over S's own TMEM columns
//   O += P V    tcgen05.mma with P read from TMEM, O (f32) in TMEM
// A tile's scores come in halves of 64 keys: one half's are there while the
// other's are turned into weights, which TMEM has no room for at 128 (S, S, O, O
// fill its 512 columns). The exponential unit needs as many cycles as the two
// products (1024 for 128 x 128 weights at 16 a cycle); a quarter of the
// exponentials go to the FMA pipe instead. Up to 128 rows there is one row tile
// and the two warpgroups take alternate key blocks, each with its own (m, sum,
// O), joined at the end.
//
//   warps 0-3, 4-7  one softmax warpgroup per tile, a thread per row: turns S
//                   into P, rescales O when the row's maximum has grown by more
//                   than 2^8 (until then the old one serves: weights stay below
//                   2^8 and the factor cancels in O / sum), writes the output or
//                   the partial result
//   warp 8          TMA: key and value blocks, page by page, into one ring
//   warps 9, 10     one per tile: issue its products (9 owns TMEM)
//   warp 11         queries of the next unit, once the last scores of this one
//                   are done with theirs
// The grid is persistent, and every role runs on into the next unit as soon as
// what it needs is there.
//
// Measured: 3 prompts of 4096 tokens, 32 query and 8 kv heads of 128, bf16, in
// 433 us (950 TFLOP/s of causal pairs) at the power cap, 375-400 us cool. No
// unit is saturated (tensor pipe 56%, exponentials 42%, issue 44%): each
// softmax warp waits on its own chain (load, maximum, exponentials, store,
// hand-over), and the clock falls to 1650 MHz. At dim 64 the compiler
// spills 48 bytes a thread.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "common.cuh"
#include "kv_half16.cuh"
#include "kv_ops.h"
#include "kv_tile_order.h"
#include "ptx.cuh"

namespace shield {
namespace kv {

using namespace tc;

// Three warpgroups. At launch every thread has 168 registers (64,512 in all);
// the two softmax warpgroups then take 224 each (half a row of S and its
// weights are 96, a row's outputs on their way out 32 more), and the third
// keeps 56: 256 * 224 + 128 * 56 = 64,512.
constexpr int TILE_THREADS = 384;
constexpr int ROWS = 128;      // rows of a tile
constexpr int BLOCK = 128;     // keys of a block, the step of the ring
constexpr int HALF = 64;       // keys of one score product: a tile's S has room for two
// One in this many pairs of weights is computed on the FMA pipe. It matters
// little while neither unit bounds the kernel (3 prompts of 4096: none 445 us,
// every 8th 445, 4th 442, 3rd 439, within a few us of one another from run to
// run); every 2nd was slower by 5%.
constexpr int POLY_EVERY = 4;
constexpr float GROWTH = 8.0f; // log2 of how far a maximum may grow before O is rescaled

template <int D>
struct TileShape {
    static constexpr int HALVES = D / 64;             // 128-byte wide operand panels
    static constexpr int PANEL = 128 * 128;           // bytes of 128 rows of one panel
    static constexpr int SLOT = HALVES * PANEL;       // a key or value block, or a row tile's queries
    static constexpr int STAGES = D == 128 ? 4 : 8;
    static constexpr int OFF_RING = 2 * SLOT;
    static constexpr int OFF_OUT = OFF_RING + STAGES * SLOT;  // 4 KB per softmax warp: outputs on their way to rows
    static constexpr int OFF_BAR = OFF_OUT + 8 * 4096;
    static constexpr int OFF_MISC = OFF_BAR + (18 + 2 * STAGES) * 8;
    static constexpr int OFF_JOIN = OFF_MISC + 16;    // (m, sum) of the second tile's rows
    static constexpr int BYTES = OFF_JOIN + ROWS * 8 + 1024;
    static_assert(ROWS * D * 4 == 2 * SLOT, "one tile's f32 outputs take the queries' place");
    static_assert(BYTES <= 227 * 1024, "shared memory per CTA");
};

// The i-th unit of this CTA: longest units first, dealt out forwards and
// backwards in turn so that every CTA gets about the same.
__device__ __forceinline__ int dealt(int i) {
    return i * (int)gridDim.x + (int)(i & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

struct TileArgs {
    AttendArgs a;
    CUtensorMap k, v;  // [layer * pages][kv head][row][dim], boxes of a page's rows by 64 dims
};

__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap *map, int x, int head, int page, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
        ::"r"(dst), "l"((uint64_t)map), "r"(x), "r"(0), "r"(head), "r"(page), "r"(bar)
        : "memory");
}

// MN-major operand (the values: dims contiguous), 128B-swizzled: panels of 64
// dims LBO apart, groups of 8 keys 1024 bytes (SBO) apart.
__device__ __forceinline__ uint64_t umma_desc_values(uint32_t saddr, uint32_t panel) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// Instruction descriptors: f32 result, 16-bit operands, M = 128.
constexpr uint32_t NEGATE_A = 1u << 13;
template <bool BF16>
constexpr uint32_t idesc_scores() {
    return (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)(HALF >> 3) << 17) | (8u << 24);
}
template <bool BF16, int D>
constexpr uint32_t idesc_values() {  // the second operand is MN-major
    return (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | (8u << 24);
}

__device__ __forceinline__ void mma_smem(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
template <uint32_t IDESC>
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "n"(IDESC), "r"(accumulate) : "memory");
}

#define R8(r, i) "=r"((r)[i]), "=r"((r)[i + 1]), "=r"((r)[i + 2]), "=r"((r)[i + 3]), "=r"((r)[i + 4]), "=r"((r)[i + 5]), "=r"((r)[i + 6]), "=r"((r)[i + 7])
#define W8(r, i) "r"((r)[i]), "r"((r)[i + 1]), "r"((r)[i + 2]), "r"((r)[i + 3]), "r"((r)[i + 4]), "r"((r)[i + 5]), "r"((r)[i + 6]), "r"((r)[i + 7])

// 32 columns of this warp's 32 TMEM lanes, a lane per thread.
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : R8(r, 0), R8(r, 8), R8(r, 16), R8(r, 24) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_load32_wait(uint32_t addr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : R8(r, 0), R8(r, 8), R8(r, 16), R8(r, 24) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
        ::W8(r, 0), W8(r, 8), W8(r, 16), W8(r, 24), "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 64 columns, defined after the wait.
__device__ __forceinline__ void tmem_load64_wait(uint32_t addr, uint32_t (&r)[64]) {
    tmem_load32(addr, r);
    tmem_load32(addr + 32, r + 32);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 64; i++) asm volatile("" : "+r"(r[i]));  // no use may move above the wait
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// The larger of three; NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// A value that is the same in the whole warp, in a form the compiler knows to
// be: operands of tcgen05.mma then stay in uniform registers.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// One lane of a converged warp.
__device__ __forceinline__ bool elected() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// One work unit as every role sees it.
struct Unit : TileOrder {
    Item it;
    int kvh;  // kv head
    __device__ __forceinline__ Unit(const AttendArgs &A, int u, uint32_t ring_) {
        it = A.plan.tile[u / A.pool.kv_heads];
        kvh = u % A.pool.kv_heads;
        const int low = it.masked ? A.plan.lim[it.tok0 + it.r0 / A.group] : it.k1;  // below it every row sees every key
        set((it.k1 - it.k0 + BLOCK - 1) / BLOCK, it.nr > ROWS, max(low - it.k0, 0) / BLOCK, ring_);
    }
};

// 2^x of a pair on the FMA pipe, for x in [-inf, 127): x = n + f with n the
// nearest integer (adding 1.5 * 2^23 + 127 leaves n + 127 in the sum's low
// bits), the polynomial that interpolates 2^f at the five Chebyshev nodes of
// [-1/2, 1/2] (at most 3.6e-6 off, over 400,001 points in f32; the weights are
// rounded to 2.4e-4 or more), times 2^n. Below -126.5 the result is 0.
__device__ __forceinline__ uint64_t exp2_poly(uint64_t x) {
    x = pack2(fmaxf(lo_f(x), -127.0f), fmaxf(hi_f(x), -127.0f));
    const uint64_t t = add2(x, pack2(12583039.0f, 12583039.0f));
    const uint64_t f = fma2(add2(t, pack2(-12583039.0f, -12583039.0f)), pack2(-1.0f, -1.0f), x);
    uint64_t p = pack2(0.00966636837f, 0.00966636837f);
    p = fma2(p, f, pack2(0.0559219755f, 0.0559219755f));
    p = fma2(p, f, pack2(0.240223497f, 0.240223497f));
    p = fma2(p, f, pack2(0.693121016f, 0.693121016f));
    p = fma2(p, f, pack2(1.0f, 1.0f));
    return mul2(p, pack2u((uint32_t)t << 23, (uint32_t)(t >> 32) << 23));
}

// Waits for a phase, 2^22 polls at most: some seconds, a poll lasting up to a
// few microseconds where it has to wait. (Watching the clock instead cost 5%.)
__device__ __forceinline__ bool arrived(uint32_t bar, uint32_t parity, volatile int *stop, int32_t *err) {
    return mbar_wait_warp<(1u << 22)>(bar, parity, stop, err);
}

template <bool BF16, int D>
__global__ void __launch_bounds__(TILE_THREADS, 1) k_attend_tile(const __grid_constant__ TileArgs args) {
    using S = TileShape<D>;
    using H = Half16<BF16>;
    // f16 weights carry a factor 2^LIFT here (with the growth, at most 2^14 in all)
    constexpr float LIFT = H::LIFT > GROWTH ? H::LIFT - GROWTH : 0.0f;
    const AttendArgs &A = args.a;
    const DevPool &P = A.pool;
    extern __shared__ uint8_t tile_smem[];
    const uint32_t base = (smem_u32(tile_smem) + 1023) & ~1023u;
    uint8_t *const smem = tile_smem + (base - smem_u32(tile_smem));
    const int warp = uniform((int)threadIdx.x >> 5), lane = threadIdx.x & 31;

    const uint32_t bars = base + S::OFF_BAR;
    const uint32_t q_full = bars, q_free = bars + 8;
    auto s_full = [&](int a, int h) { return bars + 16 + 16 * a + 8 * h; };
    auto p_full = [&](int a, int h) { return bars + 48 + 16 * a + 8 * h; };
    auto pv_done = [&](int a) { return bars + 80 + 8 * a; };  // one phase per half block
    auto o_full = [&](int a) { return bars + 96 + 8 * a; };   // one phase per unit
    const uint32_t v_clean = bars + 112;  // one phase per value block of two tiles that was looked through
    auto v_here = [&](int a) { return bars + 120 + 8 * a; };  // one phase per value block that warpgroup a looks through
    const uint32_t join_ready = bars + 136;                   // one phase per unit whose two tiles are joined
    auto full = [&](int s) { return bars + 144 + 8 * s; };
    auto empty = [&](int s) { return bars + 144 + 8 * (S::STAGES + s); };
    uint32_t *const tmem_slot = reinterpret_cast<uint32_t *>(smem + S::OFF_MISC);
    volatile int *const stop = reinterpret_cast<volatile int *>(smem + S::OFF_MISC + 4);
    volatile int *const dirty = reinterpret_cast<volatile int *>(smem + S::OFF_MISC + 8);
    float2 *const join_ml = reinterpret_cast<float2 *>(smem + S::OFF_JOIN);

    asm volatile("griddepcontrol.launch_dependents;");
    if (threadIdx.x == 0) {
        for (int a = 0; a < 2; a++) {
            for (int h = 0; h < 2; h++) {
                mbar_init(s_full(a, h), 1);
                mbar_init(p_full(a, h), 4);
            }
            mbar_init(pv_done(a), 1);
            mbar_init(v_here(a), VALUES_HERE);
            mbar_init(o_full(a), 1);
        }
        for (int s = 0; s < S::STAGES; s++) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 2);  // one per tile
        }
        mbar_init(v_clean, 4);
        mbar_init(join_ready, 2);
        mbar_init(q_full, 32);
        mbar_init(q_free, QUERIES_FREE);
        *stop = *dirty = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uniform(*tmem_slot);  // S and P of tile a's half h at 128 a + 64 h, O at 256 + 128 a

    const int units = (A.tile >= 0 ? A.tile : A.plan.counts[COUNT_TILE]) * P.kv_heads;  // the host keeps it, and one more round, below 2^31
    // No phase of a barrier may pass before all who wait for it have seen it
    // (kv_tile_order.h). What the next phase needs, barrier by barrier:
    //   q_full      both tiles' product warps; q_free, to which each of them arrives
    //               after its wait
    //   q_free      the query warp; the q_full that it tells after its wait
    //   full        both product warps; empty, to which each of them arrives
    //   empty       the copying warp; the full that it tells after its wait
    //   s_full      warpgroup a; a product that waits for all its warps' p_full
    //   p_full      product warp a; scores that it issues after its wait
    //   pv_done     warpgroup a, where a maximum grows: p_full as above
    //   v_here      the looking warpgroup; all its warps' p_full as above
    //   v_clean     tile 1's product warp; v_here, to which it arrives after its wait
    //   o_full      warpgroup a; p_full of a later unit
    //   join_ready  warpgroup 1; p_full of a later unit
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 8) {
            // ------------------------------------------------- TMA producer
            const int per = BLOCK >> P.page_shift;  // pages of a block
            uint32_t ring = 0;
            bool ok = true;
            for (int i = 0; ok && i * (int)gridDim.x < units; i++) {
                if (dealt(i) >= units) break;
                const Unit U(A, dealt(i), ring);
                // The page list in registers, a page per lane, 32 pages and the next 32,
                // so that no copy waits for its page number: `window` is the first
                // one's place among the unit's pages, at or before value block b's.
                const int32_t *const table = A.plan.table + U.it.table + (U.it.k0 >> P.page_shift);
                const int npages = (U.it.k1 - U.it.k0 + P.page_tokens - 1) >> P.page_shift;
                int window = 0;
                int here = lane < npages ? table[lane] : 0, next = 32 + lane < npages ? table[32 + lane] : 0;
                auto fill = [&](uint32_t slot, int b, const CUtensorMap *map) {
                    const int s = slot % S::STAGES;
                    const int half = lane % S::HALVES, page = lane / S::HALVES, at = b * per + page - window;
                    const int x = __shfl_sync(0xffffffffu, here, at & 31), y = __shfl_sync(0xffffffffu, next, at & 31);
                    if (!arrived(empty(s), ((slot / S::STAGES) & 1) ^ 1, stop, A.err)) return false;
                    const int pages = min(per, npages - b * per);
                    if (lane == 0) mbar_expect_tx(full(s), (uint32_t)pages * P.page_tokens * D * 2);
                    __syncwarp();
                    if (page < pages)
                        tma_load_page(base + S::OFF_RING + s * S::SLOT + half * S::PANEL + page * P.page_tokens * 128, map, half * 64,
                                      U.kvh, A.layer * P.pages + (at < 32 ? x : y), full(s));
                    return true;
                };
                for (int b = 0; ok && b < U.ahead; b++) ok = fill(U.key_slot(b), b, &args.k);
                for (int b = 0; ok && b < U.nb; b++) {
                    if (b * per - window >= 32) {
                        window += 32;
                        here = next;
                        next = window + 32 + lane < npages ? table[window + 32 + lane] : 0;
                    }
                    ok = fill(U.value_slot(b), b, &args.v);
                    if (ok && b + U.lead < U.nb) ok = fill(U.key_slot(b + U.lead), b + U.lead, &args.k);
                }
                ring += 2 * U.nb;
            }
        } else if (warp < 11) {
            // ----------------------------------------------------- products
            // The whole warp walks the schedule, so that everything in it is
            // warp-uniform, and one lane issues: with a lone thread in here the
            // descriptors have to be moved to uniform registers for each product,
            // and issuing 16 of them took longer than the tensor cores need. A wait
            // costs some 200 cycles even when its phase is complete (the products'
            // operands keep shared memory busy), so each block is waited for once,
            // and each tile has a warp of its own.
            const int a = warp - 9;
            uint32_t ring = 0, turn = 0, done = 0;  // done: key blocks of this tile in earlier units
            uint32_t cleaned = 0;                   // phases of v_clean waited for
            uint32_t seen = 0;                      // ring slots this tile has been through
            const uint32_t score_desc = idesc_scores<BF16>() | (A.scale_log2 < 0.0f ? NEGATE_A : 0u);
            const uint64_t q_desc = umma_desc_sw128(base), k_desc = umma_desc_sw128(base + S::OFF_RING);
            const uint64_t v_desc = umma_desc_values(base + S::OFF_RING, S::PANEL);
            const uint32_t st = tmem + 128 * a, ot = tmem + 256 + 128 * a;
            const bool leader = elected();
            bool ok = true;
            for (int i = 0; ok && i * (int)gridDim.x < units; i++, turn++) {
                if (dealt(i) >= units) break;
                Unit U(A, dealt(i), ring);
                U.set(uniform(U.nb), uniform(U.wide) != 0, uniform(U.clean), ring);
                const int nblocks = U.blocks_of(a), b0 = U.first_block(a), step = U.block_step();
                const uint64_t qd = q_desc + (U.wide ? a * (S::SLOT >> 4) : 0);
                // Goes through the ring up to `slot`, releasing at once what is the
                // other tile's.
                auto pass = [&](uint32_t slot) {
                    for (; seen != slot; seen++) {
                        const uint32_t s = seen % S::STAGES;
                        if (!arrived(full(s), (seen / S::STAGES) & 1, stop, A.err)) return false;
                        if (leader) mbar_arrive(empty(s));
                        __syncwarp();
                    }
                    return true;
                };
                auto filled = [&](uint32_t slot) {
                    if (!pass(slot)) return false;
                    seen++;
                    return arrived(full(slot % S::STAGES), (slot / S::STAGES) & 1, stop, A.err);
                };
                auto scores = [&](int n, int h) {  // of half h of this tile's n-th block
                    const uint32_t slot = U.key_slot(b0 + n * step), s = slot % S::STAGES;
                    if (h == 0 && !filled(slot)) return false;
                    tc_fence_after();
                    const uint64_t kd = k_desc + s * (S::SLOT >> 4) + h * (HALF * 128 >> 4);
                    if (leader) {
#pragma unroll
                        for (int i = 0; i < D / 16; i++) {
                            const uint32_t off = ((i / 4) * S::PANEL + (i % 4) * 32) >> 4;
                            mma_smem(st + 64 * h, qd + off, kd + off, score_desc, i > 0);
                        }
                        umma_commit(s_full(a, h));
                        if (h == 1) {
                            umma_commit(empty(s));
                            if (n == nblocks - 1) {
                                // The queries' place is free when both tiles and, where two
                                // warpgroups join their outputs there, these have said so.
                                for (int j = U.frees_queries(a); j > 0; j--) umma_commit(q_free);
                            }
                        }
                    }
                    __syncwarp();
                    return true;
                };
                auto values = [&](int n, int h) {
                    const uint32_t slot = U.value_slot(b0 + n * step), s = slot % S::STAGES;
                    if (h == 0 && !filled(slot)) return false;
                    const uint64_t vd = v_desc + s * (S::SLOT >> 4);
                    const bool masked = h == 0 && b0 + n * step >= U.clean;
                    if (masked && leader) mbar_arrive(v_here(U.looker(a)), U.says_values_here());
                    __syncwarp();
                    if (masked && U.wide && a == 1 && !arrived(v_clean, cleaned++ & 1, stop, A.err)) return false;
                    if (!arrived(p_full(a, h), (done + n) & 1, stop, A.err)) return false;
                    tc_fence_after();
                    if (leader) {
#pragma unroll
                        for (int i = 0; i < HALF / 16; i++)
                            mma_tmem<idesc_values<BF16, D>()>(ot, st + 64 * h + 8 * i, vd + (((4 * h + i) * 2048) >> 4), n > 0 || h > 0 || i > 0);
                        umma_commit(pv_done(a));
                        if (h == 1) {
                            umma_commit(empty(s));
                            if (n == nblocks - 1) {
                                umma_commit(o_full(a));
                                if (U.two()) umma_commit(join_ready);
                            }
                        }
                    }
                    __syncwarp();
                    return true;
                };
                ok = arrived(q_full, turn & 1, stop, A.err);
                if (nblocks > 0) ok = ok && scores(0, 0) && scores(0, 1);
                else if (ok && leader) mbar_arrive(q_free, U.frees_queries(a));
                // A half's next scores follow its weights' product, whose operand they
                // overwrite; the other half's are there already, so the softmax finds
                // scores whenever it comes back.
                for (int n = 0; ok && n < nblocks; n++) {
#pragma unroll
                    for (int h = 0; h < 2; h++) ok = ok && values(n, h) && (n + 1 >= nblocks || scores(n + 1, h));
                }
                ring += 2 * U.nb;
                ok = ok && pass(ring);
                done += nblocks;
            }
        } else {
            // ---------------------------------------------------- queries
            // 16-byte vectors to the K-major swizzled layout; rows behind the last
            // are 0.
            constexpr int VEC = D / 8, PER = 32 / VEC;  // vectors of a row, rows of one copy
            uint32_t turn = 0;
            bool ok = true;
            for (int i = 0; ok && i * (int)gridDim.x < units; i++, turn++) {
                if (dealt(i) >= units) break;
                const Unit U(A, dealt(i), 0);
                int64_t off[8];  // rows lane + 32 j
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int rr = U.it.r0 + min(lane + 32 * j, U.it.nr - 1);
                    off[j] = A.plan.perm[U.it.tok0 + rr / A.group] * A.q_stride + (U.kvh * A.group + rr % A.group) * D;
                }
                ok = arrived(q_free, (turn & 1) ^ 1, stop, A.err);
                if (!ok) break;
                const int c = lane % VEC;
                const uint32_t dst = base + (c >> 3) * S::PANEL;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    if (j >= 4 && !U.wide) break;
                    const uint32_t tile = dst + (j / 4) * S::SLOT;
#pragma unroll 8
                    for (int k = 0; k < 32; k += PER) {
                        const int r = 32 * j + k + lane / VEC;
                        const int64_t o = __shfl_sync(0xffffffffu, off[j], k + lane / VEC);
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tile + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4)),
                                     "l"(static_cast<const uint16_t *>(A.q) + o + c * 8), "r"(r < U.it.nr ? 16 : 0) : "memory");
                    }
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                fence_proxy_async();
                mbar_arrive(q_full);
            }
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int a = warp >> 2, row = threadIdx.x & 127, group = A.group;
        const float scale = fmaxf(fabsf(A.scale_log2), 1e-30f);  // a zero scale still keeps masked scores at -inf
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t st = tmem + lanes + 128 * a, ot = tmem + lanes + 256 + 128 * a;
        const uint32_t join_row = base + row * D * 4;  // 16-byte chunks xor-ed with the row against bank conflicts
        uint32_t ring = 0, turn = 0;
        uint32_t done = 0;          // key blocks of this tile in earlier units
        uint32_t ends = 0;          // earlier units in which this tile had a block
        uint32_t joins = 0;         // earlier units whose tiles were joined
        uint32_t looked = 0;        // value blocks looked through
        bool ok = true;  // false once a wait gave up: the remaining units' barriers are still met
        for (int i = 0; i * (int)gridDim.x < units; i++, turn++) {
            if (dealt(i) >= units) break;
            const Unit U(A, dealt(i), ring);
            const Item &it = U.it;
            const int r0 = it.r0 + (U.wide ? a * ROWS : 0), nr = min(ROWS, it.nr - (U.wide ? a * ROWS : 0));
            const bool live = (warp & 3) * 32 < nr;  // some row of this warp exists
            const int at = it.tok0 + min(r0 + row, r0 + nr - 1) / group;
            const int lim = row < nr ? min(it.k1, A.plan.lim[at]) : it.k1;
            // where this thread's row goes: the first byte of the output's or the partial's row
            const int rr = r0 + min(row, nr - 1);
            char *const own_row = it.part >= 0 ? reinterpret_cast<char *>(A.plan.part_o + (it.part + (int64_t)U.kvh * it.nr + (rr - it.r0)) * D)
                                               : reinterpret_cast<char *>(static_cast<uint16_t *>(A.out) + A.plan.perm[at] * A.out_stride +
                                                                          (U.kvh * group + rr % group) * D);
            float m = -INFINITY, sum = 0.0f;  // m: what the weights are relative to, in log2
            const int nblocks = U.blocks_of(a);
            for (int n = 0; ok && n < nblocks; n++) {
                const int b = U.first_block(a) + n * U.block_step(), p0 = it.k0 + b * BLOCK;
#pragma unroll 1
                for (int h = 0; h < 2; h++) {
                    if (!arrived(s_full(a, h), (done + n) & 1, stop, A.err)) {
                        ok = false;
                        break;
                    }
                    if (h == 0 && b >= U.clean && U.looker(a) == a) {
                        // Values that some row may not see must not reach its product as
                        // 0 * inf, nor may what the slot holds behind the last key: what is
                        // not finite counts as 0 here, and rows that do see such a value get it
                        // at the end.
                        const uint32_t s = U.value_slot(b) % S::STAGES;
                        if (!arrived(v_here(a), looked++ & 1, stop, A.err)) {
                            ok = false;
                            break;
                        }
                        const uint32_t values = base + S::OFF_RING + s * S::SLOT;
                        uint32_t any = 0;
#pragma unroll
                        for (int i = 0; i < S::SLOT / 16 / 128; i++) {
                            uint32_t w[4];
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                                         : "r"(values + (i * 128 + row) * 16) : "memory");
                            any |= not_finite_bits<BF16>(w[0]) | not_finite_bits<BF16>(w[1]) | not_finite_bits<BF16>(w[2]) | not_finite_bits<BF16>(w[3]);
                        }
                        if (any) {
                            bool found = false;
#pragma unroll 1
                            for (int i = row; i < S::SLOT / 16; i += 128) {
                                const bool inside = p0 + ((i * 16) % S::PANEL) / 128 < it.k1;
                                uint32_t w[4];
                                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(values + i * 16) : "memory");
                                const bool bad = (not_finite_bits<BF16>(w[0]) | not_finite_bits<BF16>(w[1]) | not_finite_bits<BF16>(w[2]) | not_finite_bits<BF16>(w[3])) != 0;
                                found |= bad && inside;
                                if (bad || !inside)
                                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(values + i * 16), "r"(inside ? finite_part<BF16>(w[0]) : 0u),
                                                 "r"(inside ? finite_part<BF16>(w[1]) : 0u), "r"(inside ? finite_part<BF16>(w[2]) : 0u),
                                                 "r"(inside ? finite_part<BF16>(w[3]) : 0u) : "memory");
                            }
                            if (found) *dirty = 1;
                        }
                        fence_proxy_async();
                        __syncwarp();
                        if (U.wide && lane == 0) mbar_arrive(v_clean);  // tile 1's products wait for it as well
                    }
                    tc_fence_after();
                    if (live) {
                        uint32_t s[HALF];
                        tmem_load64_wait(st + HALF * h, s);
                        if (b >= U.clean) {
                            const int seen = lim - p0 - HALF * h;
#pragma unroll
                            for (int i = 0; i < HALF; i++)
                                if (i >= seen) s[i] = 0xFF800000u;
                        }
                        float mx[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) mx[i] = max3(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]), -INFINITY);
#pragma unroll
                        for (int i = 8; i < HALF; i += 2) mx[(i / 2) & 3] = max3(mx[(i / 2) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                        const float top = max3(max3(mx[0], mx[1], mx[2]), mx[3], -INFINITY) * scale;
                        // also the first maximum (m is -inf before it), and a score that is not a
                        // number: m and with it the row's sum become NaN, as for one of +inf
                        const bool grown = !(top <= m + GROWTH);
                        if (__any_sync(0xffffffffu, grown)) {
                            const float f = grown ? exp2_approx(m - top) : 1.0f;
                            if (grown) m = top < INFINITY ? top : __int_as_float(0x7FC00000);
                            sum *= f;
                            if (n > 0 || h > 0) {
                                // O is still once the previous half's product is done (the one
                                // before that is: these scores came after it)
                                if (!arrived(pv_done(a), (h + 1) & 1, stop, A.err)) {
                                    ok = false;
                                    break;
                                }
                                tc_fence_after();
#pragma unroll 1
                                for (int c = 0; c < D; c += 32) {
                                    uint32_t o[32];
                                    tmem_load32_wait(ot + c, o);
#pragma unroll
                                    for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                                    tmem_store32(ot + c, o);
                                }
                            }
                        }
                        const float shift = (m == -INFINITY ? 0.0f : -m) + LIFT;
                        const uint64_t scale2 = pack2(scale, scale), shift2 = pack2(shift, shift);
                        uint64_t sum2[2] = {0, 0};
                        uint32_t w[HALF / 2];
#pragma unroll
                        for (int i = 0; i < HALF / 2; i++) {
                            const uint64_t x = fma2(pack2u(s[2 * i], s[2 * i + 1]), scale2, shift2);
                            // some on the FMA pipe: the exponential unit is the scarcer one
                            const uint64_t e = i % POLY_EVERY == POLY_EVERY - 1 ? exp2_poly(x) : pack2(exp2_approx(lo_f(x)), exp2_approx(hi_f(x)));
                            sum2[i & 1] = add2(sum2[i & 1], e);
                            w[i] = H::pack(lo_f(e), hi_f(e));
                        }
                        tmem_store32(st + HALF * h, w);
                        sum2[0] = add2(sum2[0], sum2[1]);
                        sum += lo_f(sum2[0]) + hi_f(sum2[0]);
                        tmem_store_wait();
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_full(a, h));
                }
            }
            // ---------------------------------------------------- epilogue
            if (ok && nblocks > 0) ok = arrived(o_full(a), ends & 1, stop, A.err);
            const bool two = U.two();
            if (two) {
                if (a == 1) {
                    // no product reads the queries any more once tile 0 is done too:
                    // their place takes this tile's outputs, a row a thread
                    if (ok) ok = arrived(join_ready, joins & 1, stop, A.err);
                    if (ok && live) {
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            uint32_t o[32];
                            tmem_load32_wait(ot + c, o);
#pragma unroll
                            for (int i = 0; i < 32; i += 4)
                                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(join_row + (((c + i) / 4 ^ (row & 7)) << 4)),
                                             "r"(o[i]), "r"(o[i + 1]), "r"(o[i + 2]), "r"(o[i + 3]) : "memory");
                        }
                    }
                    join_ml[row] = make_float2(m, sum);
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");
            }
            if (ok && live && (U.wide || a == 0)) {
                tc_fence_after();
                float f0 = 1.0f, f1 = 0.0f, M = m, L = sum;
                if (two) {
                    const float2 other = join_ml[row];
                    M = fmaxf(m, other.x);
                    const float ref = M == -INFINITY ? 0.0f : M;
                    f0 = exp2_approx(m - ref);
                    f1 = exp2_approx(other.x - ref);
                    L = __fmaf_rn(other.y, f1, sum * f0);
                }
                const bool mine = row < nr;
                const bool fix = *dirty != 0;  // stays set: the look is right for every unit, and only such data pays for it
                const int64_t part = it.part + (int64_t)U.kvh * it.nr + (r0 - it.r0);
                const float inv = it.part < 0 ? 1.0f / L : 1.0f;
                // partials of the few-row kernel carry 2^H::LIFT: say the same of these
                if (mine && it.part >= 0) A.plan.part_ml[part + row] = make_float2(M + (H::LIFT - LIFT), L);
                // A thread holds a row; rows go out through shared memory (128 bytes of
                // each at a time, 16-byte chunks xor-ed with the row against bank
                // conflicts), so that 8 lanes write 128 bytes of one row together
                // instead of 32 lanes 16 bytes of 32 rows.
                const uint32_t stage = base + S::OFF_OUT + warp * 4096;
                auto flush = [&](int byte) {
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int r = (lane >> 3) + 4 * j;
                        uint32_t w[4];
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                                     : "r"(stage + r * 128 + (((lane & 7) ^ (r & 7)) << 4)) : "memory");
                        char *const to = reinterpret_cast<char *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(own_row), r));
                        if ((warp & 3) * 32 + r < nr) *reinterpret_cast<uint4 *>(to + byte + (lane & 7) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    __syncwarp();
                };
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    tmem_load32_wait(ot + c, o);
                    if (two) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            float y[4];
                            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(y[0]), "=f"(y[1]), "=f"(y[2]), "=f"(y[3])
                                         : "r"(join_row + (((c + j) / 4 ^ (row & 7)) << 4)) : "memory");
#pragma unroll
                            for (int k = 0; k < 4; k++) o[j + k] = __float_as_uint(__fmaf_rn(y[k], f1, __uint_as_float(o[j + k]) * f0));
                        }
                    }
                    if (fix && mine) {
                        const int32_t *const table = A.plan.table + it.table;
#pragma unroll 1
                        for (int p = it.k0 + U.clean * BLOCK; p < lim; p++) {
                            const uint16_t *v = static_cast<const uint16_t *>(P.v) +
                                row_offset(P, A.layer, table[p >> P.page_shift], U.kvh, p & (P.page_tokens - 1)) + c;
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                if ((v[j] & H::EXP) == H::EXP) o[j] = __float_as_uint(__uint_as_float(o[j]) + H::value(v[j]));
                        }
                    }
                    auto put = [&](int chunk, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128 + ((chunk ^ (lane & 7)) << 4)), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
                    };
                    if (it.part < 0) {  // two column groups of 32 make 128 bytes
#pragma unroll
                        for (int j = 0; j < 32; j += 8) {
                            uint32_t w[4];
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                w[k] = H::pack(__uint_as_float(o[j + 2 * k]) * inv, __uint_as_float(o[j + 2 * k + 1]) * inv);
                            put((c & 32) / 8 + j / 8, w[0], w[1], w[2], w[3]);
                        }
                        if (c & 32) flush((c - 32) * 2);
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j += 4) put(j / 4, o[j], o[j + 1], o[j + 2], o[j + 3]);
                        flush(c * 4);
                    }
                }
            }
            tc_fence_before();
            ring += 2 * U.nb;
            done += nblocks;
            ends += nblocks > 0;
            joins += two;
            if (two) {  // the joined outputs have been read: their place is free
                asm volatile("bar.sync 2, 256;" ::: "memory");
                if (threadIdx.x == 0) mbar_arrive(q_free);
            }
        }
    }
    __syncthreads();
    // After a wait gave up, copies and products may still be on their way: give
    // them a bounded time before the memory they use is let go.
    if (*stop) {
        const long long t0 = clock64();
        while (clock64() - t0 < 400000000LL) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// ------------------------------------------------------------------ host

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    if (!fn) {
        cudaDriverEntryPointQueryResult q;
        void *p = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }
    return fn;
}

bool map_pool(CUtensorMap *m, const DevPool &P, void *data) {
    auto fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t row = (cuuint64_t)P.dim * 2;
    cuuint64_t dims[4] = {(cuuint64_t)P.dim, (cuuint64_t)P.page_tokens, (cuuint64_t)P.kv_heads, (cuuint64_t)P.layers * P.pages};
    cuuint64_t strides[3] = {row, row * P.page_tokens, row * P.page_tokens * P.kv_heads};
    cuuint32_t box[4] = {64, (cuuint32_t)P.page_tokens, 1, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    return fn(m, P.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, data, dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool BF16, int D>
static cudaError_t tile_launch(const TileArgs &T, int64_t units, int sms, cudaStream_t s) {
    using S = TileShape<D>;
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t e = allow_smem(k_attend_tile<BF16, D>, S::BYTES, allowed);
    if (e != cudaSuccess) return e;
    return launch(k_attend_tile<BF16, D>, (unsigned)std::min<int64_t>(units, sms), TILE_THREADS, S::BYTES, false, s, T);
}

cudaError_t launch_attend_tile(const AttendArgs &A, const CUtensorMap *maps, int64_t units, int sms, cudaStream_t s) {
    if (units == 0) return cudaSuccess;
    TileArgs T;
    T.a = A;
    T.k = maps[0];
    T.v = maps[1];
    if (A.pool.dim == 128) return A.pool.bf16 ? tile_launch<true, 128>(T, units, sms, s) : tile_launch<false, 128>(T, units, sms, s);
    if (A.pool.dim == 64) return A.pool.bf16 ? tile_launch<true, 64>(T, units, sms, s) : tile_launch<false, 64>(T, units, sms, s);
    return cudaErrorInvalidValue;
}

}  // namespace kv
}  // namespace shield
