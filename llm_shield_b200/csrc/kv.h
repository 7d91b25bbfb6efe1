// Paged key/value caches of a context: the pools, their sequences and the
// batches whose plans the attention reads.
#pragma once

#include <memory>
#include <unordered_map>
#include <vector>

#include "context.h"
#include "kv_ops.h"

namespace shield {
namespace kv {

struct Batch;

struct Cache {
    int64_t id = 0;
    DeviceView dev;
    DevPool pool;
    CUtensorMap maps[2];  // keys, values
    Pool book;
    int32_t device = 0;  // index within the context
    bool owns = false;   // the pool's memory is the library's
    std::unique_ptr<Batch> model;  // of the model's own forwards
    explicit Cache(const Pool &b) : book(b) {}
    ~Cache();
};

struct Batch {
    Cache *cache = nullptr;
    int32_t n_heads = 0, max_tokens = 0, max_seqs = 0, max_positions = 0;
    PlanShape shape;
    char *dev = nullptr;                 // every array of the plan at a fixed offset, then the partials
    char *host[2] = {nullptr, nullptr};  // pinned images of the plan, used in turn (one allocation)
    cudaEvent_t sent[2] = {nullptr, nullptr};
    int turn = 0;
    size_t bytes = 0;             // of the plan
    int32_t *err = nullptr;       // error word of the kernels' bounded waits, in mapped host memory
    DevPlan plan;
    Plan last;                    // what was uploaded
    std::vector<int64_t> seqs;    // the sequences it covers
    int64_t frees = 0, moves = 0; // the pool's counts when it was planned
    bool planned = false;
    bool meets = false;           // two sequences hold a position of the step in common
    ~Batch();
};

// The cache's batch for the model's own forwards, with room for a step of this
// size: made anew, once the GPU is done with it, when it has to grow, and then
// with room for more, up to steps of most_tokens and sequences of most_positions.
Batch &model_batch(Cache &c, int32_t n_heads, int32_t tokens, int32_t seqs, int32_t positions, int32_t most_tokens, int32_t most_positions);
// Plans a step on the context's stream; the calls below are one layer of it.
void set_batch(Batch &B, const int64_t *seqs, const int32_t *counts, int32_t n, cudaStream_t s);
void write_layer(Batch &B, int32_t layer, const float *k, const float *v, cudaStream_t s);
void attend_layer(Batch &B, int32_t layer, const void *q, void *out, float scale, cudaStream_t s);
// Throws when a wait of the batch's finished work gave up.
void check_error(Batch &B);
Cache &cache_of(shield_ctx *ctx, int64_t id);

struct State {
    int64_t next_cache = 1, next_batch = 1;
    std::unordered_map<int64_t, std::unique_ptr<Cache>> caches;
    std::unordered_map<int64_t, std::unique_ptr<Batch>> batches;  // destroyed before the caches
    ~State() { batches.clear(); }
};

}  // namespace kv
}  // namespace shield
