// The order of one work unit of the many-row attention kernel
// (kv_attn_tile.cu): which ring slots its blocks take, which blocks each row
// tile computes, and how often each role arrives on the barriers that several
// roles share. Host and device, no CUDA: tests run the roles through it with
// unequal speeds.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define SHIELD_HD __host__ __device__ __forceinline__
#else
#define SHIELD_HD inline
#endif

namespace shield {
namespace kv {

// A barrier only tells the parity of its phase: a phase that completes before
// the one before it has been seen by everyone who waits for it looks as if it
// had not completed, and the wait runs out. So whoever waits on a barrier waits
// for each of its phases in turn, and what completes a phase comes, directly or
// through others, after everyone has seen the last.
constexpr int VALUES_HERE = 2;   // arrivals on v_here per phase
constexpr int QUERIES_FREE = 3;  // arrivals on q_free per phase

struct TileOrder {
    int nb = 0;               // key blocks
    bool wide = false;        // two row tiles; else one, whose two warpgroups take alternate key blocks
    int lead = 2, ahead = 0;  // key blocks whose scores run ahead of their weights, and how many there are
    int clean = 0;            // whole key blocks that no row is masked in
    uint32_t ring = 0;        // ring slots filled by earlier units

    SHIELD_HD void set(int nb_, bool wide_, int clean_, uint32_t ring_) {
        nb = nb_;
        wide = wide_;
        lead = wide ? 1 : 2;
        ahead = lead < nb ? lead : nb;
        clean = clean_;
        ring = ring_;
    }
    // The ring's order: the first `ahead` key blocks, then value block i
    // followed by key block i + lead while there is one.
    SHIELD_HD uint32_t key_slot(int b) const { return ring + (b < ahead ? b : ahead + 2 * (b - lead) + 1); }
    SHIELD_HD uint32_t value_slot(int b) const { return ring + ahead + b + (b < nb - ahead ? b : nb - ahead); }
    SHIELD_HD bool two() const { return !wide && nb > 1; }  // both warpgroups hold part of the same rows
    SHIELD_HD int blocks_of(int tile) const { return wide ? nb : (nb - tile + 1) / 2; }
    SHIELD_HD int first_block(int tile) const { return wide ? 0 : tile; }
    SHIELD_HD int block_step() const { return wide ? 1 : 2; }

    // The warpgroup that looks through the value blocks that a tile multiplies.
    SHIELD_HD int looker(int tile) const { return wide ? 0 : tile; }
    // Arrivals of a tile's product warp on its looker's v_here for a masked block.
    // Of two tiles each gives one, so the looker cannot finish a second block
    // (v_clean) before tile 1's product warp has waited for the first.
    SHIELD_HD int says_values_here() const { return wide ? 1 : VALUES_HERE; }
    // Arrivals of a tile's product warp on q_free: with the commit of its last
    // scores or, where it has no block, as soon as it has waited for the queries
    // (q_full), so that the next unit's cannot come before it has seen these. The
    // third of two() is the softmax's, when the joined outputs have been read.
    SHIELD_HD int frees_queries(int tile) const { return blocks_of(tile) == 0 ? 1 : wide ? 1 + tile : two() ? 1 : 2; }
};

}  // namespace kv
}  // namespace shield
