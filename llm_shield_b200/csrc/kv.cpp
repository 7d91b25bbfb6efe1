// C ABI of the paged key/value caches (include/shield_b200.h).
#include <algorithm>
#include <cmath>
#include <cstring>
#include <unordered_set>

#include "kv.h"
#include "ops.h"

namespace shield {
namespace kv {

Cache::~Cache() {
    model.reset();
    if (!owns) return;
    int before = -1;
    cudaGetDevice(&before);
    cudaSetDevice(dev.ordinal);
    cudaFree(pool.k);
    cudaFree(pool.v);
    if (before >= 0) cudaSetDevice(before);
}

Batch::~Batch() {
    int before = -1;
    cudaGetDevice(&before);
    if (cache) cudaSetDevice(cache->dev.ordinal);
    for (int i = 0; i < 2; i++) {
        if (sent[i]) {
            cudaEventSynchronize(sent[i]);
            cudaEventDestroy(sent[i]);
        }
    }
    if (host[0]) cudaFreeHost(host[0]);
    cudaFree(dev);
    if (before >= 0) cudaSetDevice(before);
}

Cache &cache_of(shield_ctx *ctx, int64_t id) {
    if (!ctx) throw Error(SHIELD_ERR_ARG, "ctx is null");
    State &S = kv_state(ctx);
    auto it = S.caches.find(id);
    if (it == S.caches.end()) throw Error(SHIELD_ERR_ARG, "unknown cache " + std::to_string(id));
    return *it->second;
}

static Batch &batch_of(shield_ctx *ctx, int64_t id) {
    if (!ctx) throw Error(SHIELD_ERR_ARG, "ctx is null");
    State &S = kv_state(ctx);
    auto it = S.batches.find(id);
    if (it == S.batches.end()) throw Error(SHIELD_ERR_ARG, "unknown batch " + std::to_string(id));
    return *it->second;
}

static cudaStream_t stream_of(const Cache &c, void *stream) {
    return stream ? static_cast<cudaStream_t>(stream) : c.dev.stream;
}

static bool capturing(cudaStream_t s) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    SHIELD_CUDA(cudaStreamIsCapturing(s, &st));
    return st != cudaStreamCaptureStatusNone;
}

// Calls that change the bookkeeping happen once, at the call: a captured copy
// of their kernels would be replayed without it.
static void not_captured(cudaStream_t s, const char *what) {
    if (capturing(s)) throw Error(SHIELD_ERR_STATE, std::string(what) + " cannot be captured into a graph");
}

static void check(cudaError_t e, const char *what) {
    if (e == cudaSuccess) return;
    cudaGetLastError();
    throw Error(SHIELD_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

static void need(int32_t n, const void *p, const char *what) {
    if (n < 0) throw Error(SHIELD_ERR_ARG, "negative count");
    if (n > 0 && !p) throw Error(SHIELD_ERR_ARG, std::string(what) + " is null");
}

static void create(shield_ctx *ctx, int32_t device, const shield_kv_config *cfg, int64_t *out) {
    if (!ctx || !cfg || !out) throw Error(SHIELD_ERR_ARG, "null argument");
    const shield_kv_config &c = *cfg;
    if (c.type != SHIELD_TYPE_F16 && c.type != SHIELD_TYPE_BF16)
        throw Error(SHIELD_ERR_UNSUPPORTED, "a paged cache holds F16 or BF16");
    if (c.n_layers <= 0 || c.n_kv_heads <= 0 || c.n_pages <= 0) throw Error(SHIELD_ERR_ARG, "every size must be positive");
    if (c.head_dim != 64 && c.head_dim != 128) throw Error(SHIELD_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
    if (c.page_tokens != 16 && c.page_tokens != 32 && c.page_tokens != 64 && c.page_tokens != 128)
        throw Error(SHIELD_ERR_UNSUPPORTED, "page_tokens must be 16, 32, 64 or 128");
    if ((int64_t)c.n_pages * c.page_tokens > INT32_MAX || c.n_layers > 4096 || c.n_kv_heads > 1024)
        throw Error(SHIELD_ERR_RANGE, "the pool is too large");
    if (!c.k != !c.v) throw Error(SHIELD_ERR_ARG, "k and v are both given or both null");
    if ((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) % 128)
        throw Error(SHIELD_ERR_ARG, "k and v must start on 128-byte boundaries");
    const DeviceView dev = device_view(ctx, device);
    DeviceScope scope(dev.ordinal);
    State &S = kv_state(ctx);
    const int64_t id = S.next_cache;
    if (id >= 1 << 18) throw Error(SHIELD_ERR_RANGE, "the context has made too many caches");  // ids hold 18 bits of it
    auto cache = std::make_unique<Cache>(Pool(c.n_pages, c.page_tokens, id));
    cache->id = id;
    cache->dev = dev;
    cache->device = device;
    DevPool &P = cache->pool;
    P.bf16 = c.type == SHIELD_TYPE_BF16;
    P.layers = c.n_layers;
    P.pages = c.n_pages;
    P.kv_heads = c.n_kv_heads;
    P.page_tokens = c.page_tokens;
    P.page_shift = c.page_tokens == 16 ? 4 : c.page_tokens == 32 ? 5 : c.page_tokens == 64 ? 6 : 7;
    P.dim = c.head_dim;
    if (c.k) {
        P.k = c.k;
        P.v = c.v;
    } else {
        cache->owns = true;  // what has been allocated is freed if the next line fails
        SHIELD_CUDA(cudaMalloc(&P.k, (size_t)P.layer_stride() * P.layers * 2));
        SHIELD_CUDA(cudaMalloc(&P.v, (size_t)P.layer_stride() * P.layers * 2));
    }
    if (!map_pool(&cache->maps[0], P, P.k) || !map_pool(&cache->maps[1], P, P.v))
        throw Error(SHIELD_ERR_CUDA, "the pool's memory cannot be mapped for TMA");
    S.caches.emplace(id, std::move(cache));
    S.next_cache++;
    *out = id;
}

static void fork(shield_ctx *ctx, int64_t kv, const int64_t *seqs, const int32_t *lens, int32_t n, int64_t *out,
                 bool share, void *stream) {
    Cache &c = cache_of(ctx, kv);
    need(n, seqs, "seqs");
    need(n, out, "out");
    if (n == 0) return;
    DeviceScope scope(c.dev.ordinal);
    const cudaStream_t s = stream_of(c, stream);
    not_captured(s, share ? "a fork" : "a copy");
    std::vector<Move> moves;
    std::vector<int64_t> ids((size_t)n);  // seqs and out may be the same array
    c.book.fork(seqs, lens, n, share, ids.data(), moves);
    const cudaError_t e = launch_move_pages(c.pool, moves.data(), (int64_t)moves.size(), s);
    if (e != cudaSuccess) {
        c.book.free(ids.data(), n);
        check(e, "copying pages");
    }
    std::copy(ids.begin(), ids.end(), out);
}

static std::unique_ptr<Batch> make_batch(Cache &c, const shield_kv_batch_config *cfg) {
    if (cfg->n_heads <= 0 || cfg->n_heads % c.pool.kv_heads)
        throw Error(SHIELD_ERR_SHAPE, std::to_string(cfg->n_heads) + " query heads do not divide into " +
                                          std::to_string(c.pool.kv_heads) + " kv heads");
    if (cfg->max_tokens <= 0 || cfg->max_seqs <= 0 || cfg->max_positions <= 0)
        throw Error(SHIELD_ERR_ARG, "every capacity must be positive");
    DeviceScope scope(c.dev.ordinal);
    auto B = std::make_unique<Batch>();
    B->cache = &c;
    B->n_heads = cfg->n_heads;
    B->max_tokens = cfg->max_tokens;
    B->max_seqs = cfg->max_seqs;
    B->max_positions = cfg->max_positions;
    PlanShape &S = B->shape;
    const int64_t T = cfg->max_tokens, n = cfg->max_seqs;
    S.group = cfg->n_heads / c.pool.kv_heads;
    S.kv_heads = c.pool.kv_heads;
    S.sms = c.dev.sms;
    S.max_items = 2 * (n + (T * S.group + FEW_TILE - 1) / FEW_TILE) + 4096;
    S.max_segments = 2 * n;
    S.max_part = std::min<int64_t>(262144, 16 * T * cfg->n_heads + 16384);
    S.max_table = n * ((cfg->max_positions + (int64_t)c.pool.page_tokens - 1) / c.pool.page_tokens);
    // (the kernels count items times kv heads, and a round beyond, in 32 bits)
    if (T * S.group > (1 << 30) || S.max_table > (1 << 30) || S.max_items * S.kv_heads > (1 << 30))
        throw Error(SHIELD_ERR_RANGE, "the batch is too large");
    size_t at = 0;
    auto place = [&](size_t count, size_t size) {
        const size_t p = at;
        at = (at + count * size + 127) / 128 * 128;
        return p;
    };
    const size_t o_counts = place(COUNTS, 4), o_few = place((size_t)S.max_items, sizeof(Item)),
                 o_tile = place((size_t)S.max_items, sizeof(Item)), o_segs = place((size_t)S.max_segments, sizeof(Segment)),
                 o_slot = place((size_t)T, 4), o_perm = place((size_t)T, 4), o_lim = place((size_t)T, 4),
                 o_merge = place((size_t)T, sizeof(Join)), o_where = place((size_t)S.max_items, 4),
                 o_table = place((size_t)S.max_table, 4);
    B->bytes = at;
    const size_t o_part = place((size_t)S.max_part * c.pool.dim, 4), o_ml = place((size_t)S.max_part, sizeof(float2));
    SHIELD_CUDA(cudaMalloc(&B->dev, at));
    // two images of the plan, and the error word
    SHIELD_CUDA(cudaHostAlloc(reinterpret_cast<void **>(&B->host[0]), 2 * B->bytes + 4, cudaHostAllocMapped));
    B->host[1] = B->host[0] + B->bytes;
    B->err = reinterpret_cast<int32_t *>(B->host[0] + 2 * B->bytes);
    *B->err = 0;
    for (auto &e : B->sent) SHIELD_CUDA(cudaEventCreateWithFlags(&e, cudaEventDisableTiming));
    // (nothing is launched on the plan's memory before a plan is set)
    auto ints = [&](size_t o) { return reinterpret_cast<const int32_t *>(B->dev + o); };
    DevPlan &P = B->plan;
    P.counts = ints(o_counts);
    P.few = reinterpret_cast<const Item *>(B->dev + o_few);
    P.tile = reinterpret_cast<const Item *>(B->dev + o_tile);
    P.segs = reinterpret_cast<const Segment *>(B->dev + o_segs);
    P.slot = ints(o_slot);
    P.perm = ints(o_perm);
    P.lim = ints(o_lim);
    P.merge = reinterpret_cast<const Join *>(B->dev + o_merge);
    P.where = ints(o_where);
    P.table = ints(o_table);
    P.part_o = reinterpret_cast<float *>(B->dev + o_part);
    P.part_ml = reinterpret_cast<float2 *>(B->dev + o_ml);
    return B;
}

static void batch_create(shield_ctx *ctx, int64_t kv, const shield_kv_batch_config *cfg, int64_t *out) {
    Cache &c = cache_of(ctx, kv);
    if (!cfg || !out) throw Error(SHIELD_ERR_ARG, "null argument");
    auto B = make_batch(c, cfg);
    State &st = kv_state(ctx);
    *out = st.next_batch++;
    st.batches.emplace(*out, std::move(B));
}

Batch &model_batch(Cache &c, int32_t n_heads, int32_t tokens, int32_t seqs, int32_t positions, int32_t most_tokens, int32_t most_positions) {
    Batch *b = c.model.get();
    if (b && b->n_heads == n_heads && b->max_tokens >= tokens && b->max_seqs >= seqs && b->max_positions >= positions) return *b;
    const bool grows = b && b->n_heads == n_heads;
    // (a step has no more sequences than tokens)
    const shield_kv_batch_config need{n_heads, tokens, seqs, positions},
        roomy{n_heads, grown(grows ? b->max_tokens : 0, tokens, most_tokens), grown(grows ? b->max_seqs : 0, seqs, most_tokens),
              grown(grows ? b->max_positions : 0, positions, most_positions)};
    SHIELD_CUDA(cudaStreamSynchronize(c.dev.stream));
    c.model.reset();
    try {
        c.model = make_batch(c, &roomy);
    } catch (const Error &) {  // no memory for that much
        c.model = make_batch(c, &need);
    }
    return *c.model;
}

// The kernels' bounded waits report here; the host sees it at the next call.
void check_error(Batch &B) {
    const int32_t e = *static_cast<volatile int32_t *>(B.err);
    if (!e) return;
    *B.err = 0;
    throw Error(SHIELD_ERR_TIMEOUT, "a device-side wait of an earlier call gave up (error word " + std::to_string(e) + ")");
}

void set_batch(Batch &B, const int64_t *seqs, const int32_t *counts, int32_t n, cudaStream_t s) {
    Cache &c = *B.cache;
    check_error(B);
    if (n > B.max_seqs)
        throw Error(SHIELD_ERR_RANGE, std::to_string(n) + " sequences, more than max_seqs " + std::to_string(B.max_seqs));
    int64_t tokens = 0;
    std::unordered_set<int64_t> seen;
    for (int32_t i = 0; i < n; i++) {
        const Sequence &s = c.book.get(seqs[i]);
        if (!seen.insert(seqs[i]).second)
            throw Error(SHIELD_ERR_ARG, "sequence " + std::to_string(seqs[i]) + " appears twice in one call");
        if (counts[i] < 0 || counts[i] > s.len)
            throw Error(SHIELD_ERR_RANGE, "sequence " + std::to_string(seqs[i]) + " holds " + std::to_string(s.len) +
                                              " positions, not " + std::to_string(counts[i]));
        if (s.len > B.max_positions)
            throw Error(SHIELD_ERR_RANGE, "sequence " + std::to_string(seqs[i]) + " holds " + std::to_string(s.len) +
                                              " positions, more than max_positions " + std::to_string(B.max_positions));
        tokens += counts[i];
    }
    if (tokens > B.max_tokens)
        throw Error(SHIELD_ERR_RANGE, std::to_string(tokens) + " tokens, more than max_tokens " + std::to_string(B.max_tokens));
    DeviceScope scope(c.dev.ordinal);
    not_captured(s, "setting a batch");
    Plan plan;
    make_plan(c.book, seqs, counts, n, B.shape, plan);
    const int turn = B.turn;
    SHIELD_CUDA(cudaEventSynchronize(B.sent[turn]));  // the upload two calls ago has left this image
    char *h = B.host[turn];
    B.planned = false;
    auto send = [&](const void *dev, const void *src, size_t bytes) {
        if (!bytes) return;
        const size_t o = (size_t)(static_cast<const char *>(dev) - B.dev);
        memcpy(h + o, src, bytes);
        SHIELD_CUDA(cudaMemcpyAsync(B.dev + o, h + o, bytes, cudaMemcpyHostToDevice, s));
    };
    const int32_t count[COUNTS] = {(int32_t)tokens, (int32_t)plan.few.size(), (int32_t)plan.tile.size(), (int32_t)plan.merge.size(), plan.solo};
    const DevPlan &P = B.plan;
    send(P.counts, count, sizeof(count));
    send(P.few, plan.few.data(), plan.few.size() * sizeof(Item));
    send(P.tile, plan.tile.data(), plan.tile.size() * sizeof(Item));
    send(P.segs, plan.segs.data(), plan.segs.size() * sizeof(Segment));
    send(P.slot, plan.slot.data(), plan.slot.size() * 4);
    send(P.perm, plan.perm.data(), plan.perm.size() * 4);
    send(P.lim, plan.lim.data(), plan.lim.size() * 4);
    send(P.merge, plan.merge.data(), plan.merge.size() * sizeof(Join));
    send(P.where, plan.where.data(), plan.where.size() * 4);
    send(P.table, plan.table.data(), plan.table.size() * 4);
    SHIELD_CUDA(cudaEventRecord(B.sent[turn], s));
    B.turn ^= 1;
    B.last = std::move(plan);
    B.seqs.assign(seqs, seqs + n);
    B.frees = c.book.frees();
    B.moves = c.book.moves();
    B.meets = steps_meet(c.book, seqs, counts, n);
    B.planned = true;
}

static void batch_set(shield_ctx *ctx, int64_t batch, const int64_t *seqs, const int32_t *counts, int32_t n, void *stream) {
    Batch &B = batch_of(ctx, batch);
    need(n, seqs, "seqs");
    need(n, counts, "counts");
    set_batch(B, seqs, counts, n, stream_of(*B.cache, stream));
}

// A plan holds while its sequences live and no page has moved.
static void check_plan(Batch &B) {
    check_error(B);
    if (!B.planned) throw Error(SHIELD_ERR_STATE, "the batch has no plan (shield_kv_batch_set)");
    const Pool &book = B.cache->book;
    if (B.moves != book.moves()) throw Error(SHIELD_ERR_STATE, "pages have moved since the batch was set");
    if (B.frees != book.frees()) {
        for (int64_t id : B.seqs)
            if (!book.has(id)) throw Error(SHIELD_ERR_STATE, "a sequence of the batch has been freed");
        B.frees = book.frees();
    }
}

static void check_layer(const Cache &c, int32_t layer) {
    if (layer < 0 || layer >= c.pool.layers)
        throw Error(SHIELD_ERR_RANGE, "layer " + std::to_string(layer) + " is outside the cache's " + std::to_string(c.pool.layers));
}

// Rows of `width` elements, `stride` apart (0: packed); 16-byte vectors.
static int64_t row_stride(int64_t stride, int64_t width, const void *p, int elt, const char *what) {
    if (!p) throw Error(SHIELD_ERR_ARG, std::string(what) + " is null");
    if (stride == 0) stride = width;
    if (stride < width) throw Error(SHIELD_ERR_ARG, std::string(what) + ": rows overlap (stride " + std::to_string(stride) + " < " + std::to_string(width) + ")");
    if (reinterpret_cast<uintptr_t>(p) % 16 || stride * elt % 16)
        throw Error(SHIELD_ERR_ARG, std::string(what) + ": rows must start on 16-byte boundaries");
    return stride;
}

// Whether some of `tokens` output rows may lie over the queries of another token
// or head: not where the two are one array, lie apart, or take turns in rows of
// one stride.
static bool rows_clash(const void *q, int64_t q_stride, const void *out, int64_t out_stride, int64_t width, int64_t tokens) {
    if (tokens == 0 || (q == out && (tokens == 1 || q_stride == out_stride))) return false;
    const int64_t a = (int64_t)reinterpret_cast<uintptr_t>(q), b = (int64_t)reinterpret_cast<uintptr_t>(out);
    const int64_t a_end = a + ((tokens - 1) * q_stride + width) * 2, b_end = b + ((tokens - 1) * out_stride + width) * 2;
    if (a_end <= b || b_end <= a) return false;
    if (q_stride != out_stride) return true;
    const int64_t row = q_stride * 2, off = ((b - a) % row + row) % row;
    return off < width * 2 || off > row - width * 2;
}

static void write_rows(Batch &B, int32_t layer, uint32_t type, const void *k, int64_t k_stride, const void *v,
                       int64_t v_stride, cudaStream_t s) {
    Cache &c = *B.cache;
    check_plan(B);
    check_layer(c, layer);
    if (B.meets) throw Error(SHIELD_ERR_STATE, "two sequences of the batch share a position of the step: their rows would be written to one place");
    if (type != SHIELD_TYPE_F32 && type != (c.pool.bf16 ? SHIELD_TYPE_BF16 : SHIELD_TYPE_F16))
        throw Error(SHIELD_ERR_UNSUPPORTED, "rows are F32 or of the cache's own type");
    const int64_t width = (int64_t)c.pool.kv_heads * c.pool.dim;
    const int elt = type == SHIELD_TYPE_F32 ? 4 : 2;
    DeviceScope scope(c.dev.ordinal);
    const bool cap = capturing(s);
    const int64_t tokens = cap ? B.max_tokens : (int64_t)B.last.slot.size();
    if (tokens == 0) return;
    k_stride = row_stride(k_stride, width, k, elt, "k");
    v_stride = row_stride(v_stride, width, v, elt, "v");
    check(launch_write_rows(c.pool, B.plan, tokens, layer, elt == 4, k, k_stride, v, v_stride, s), "writing rows");
}

static void attend(Batch &B, int32_t layer, const void *q, int64_t q_stride, void *out, int64_t out_stride, float scale,
                   cudaStream_t s) {
    Cache &c = *B.cache;
    check_plan(B);
    check_layer(c, layer);
    if (!std::isfinite(scale)) throw Error(SHIELD_ERR_ARG, "scale must be finite");
    const int64_t width = (int64_t)B.n_heads * c.pool.dim;
    DeviceScope scope(c.dev.ordinal);
    AttendArgs A;
    const bool cap = capturing(s);
    if (!cap && B.last.perm.empty()) return;
    A.q_stride = row_stride(q_stride, width, q, 2, "q");
    A.out_stride = row_stride(out_stride, width, out, 2, "out");
    // (captured: later plans' tokens are not known, so only what clashes from two on)
    if (cap ? q == out && A.q_stride != A.out_stride && B.max_tokens > 1
            : rows_clash(q, A.q_stride, out, A.out_stride, width, (int64_t)B.last.perm.size()))
        throw Error(SHIELD_ERR_ARG, "out overlaps q (it may be q, with q's stride)");
    A.pool = c.pool;
    A.plan = B.plan;
    A.q = q;
    A.out = out;
    A.layer = layer;
    A.group = B.shape.group;
    A.scale_log2 = scale * 1.44269504088896340736f;
    A.err = B.err;
    if (!cap) {
        A.few = (int32_t)B.last.few.size();
        A.solo = B.last.solo;
        A.tile = (int32_t)B.last.tile.size();
    }
    // A captured launch replays whatever plan is set then: enough CTAs for any,
    // each striding over the plan's own count.
    const int64_t alone = (int64_t)B.last.solo * c.pool.kv_heads;
    const int64_t few = cap ? 2 * (int64_t)c.dev.sms : (int64_t)B.last.few.size() * c.pool.kv_heads - alone + (alone + 3) / 4;
    const int64_t tile = cap ? (int64_t)c.dev.sms : (int64_t)B.last.tile.size() * c.pool.kv_heads;
    const int64_t join = cap ? std::min<int64_t>(B.max_tokens, 4096) : (int64_t)B.last.merge.size();
    check(launch_attend_tile(A, c.maps, tile, c.dev.sms, s), "attention, many rows");
    check(launch_attend_few(A, few, tile > 0, s), "attention, few rows");
    check(launch_attend_merge(A, join, s), "attention, joining");
}

void write_layer(Batch &B, int32_t layer, const float *k, const float *v, cudaStream_t s) {
    write_rows(B, layer, SHIELD_TYPE_F32, k, 0, v, 0, s);
}

void attend_layer(Batch &B, int32_t layer, const void *q, void *out, float scale, cudaStream_t s) {
    attend(B, layer, q, 0, out, 0, scale, s);
}

}  // namespace kv
}  // namespace shield

using namespace shield;

extern "C" {

shield_status shield_kv_create(shield_ctx *ctx, int32_t device, const shield_kv_config *cfg, int64_t *kv) {
    return guarded([&] { kv::create(ctx, device, cfg, kv); });
}

shield_status shield_kv_release(shield_ctx *ctx, int64_t kv) {
    return guarded([&] {
        kv::Cache &c = kv::cache_of(ctx, kv);
        kv::State &S = kv_state(ctx);
        DeviceScope scope(c.dev.ordinal);
        for (auto it = S.batches.begin(); it != S.batches.end();) {
            if (it->second->cache == &c) it = S.batches.erase(it);
            else ++it;
        }
        S.caches.erase(kv);
    });
}

shield_status shield_kv_get_info(shield_ctx *ctx, int64_t kv, shield_kv_info *out) {
    return guarded([&] {
        kv::Cache &c = kv::cache_of(ctx, kv);
        if (!out) throw Error(SHIELD_ERR_ARG, "out is null");
        shield_kv_info i{};
        i.n_pages = c.book.n_pages();
        i.pages_used = c.book.pages_used();
        i.pages_spanned = c.book.pages_spanned();
        i.n_seqs = c.book.sequences();
        i.page_tokens = c.pool.page_tokens;
        i.k = c.pool.k;
        i.v = c.pool.v;
        *out = i;
    });
}

shield_status shield_kv_open(shield_ctx *ctx, int64_t kv, int32_t n, int64_t *seqs) {
    return guarded([&] {
        kv::Cache &c = kv::cache_of(ctx, kv);
        kv::need(n, seqs, "seqs");
        c.book.open(n, seqs);
    });
}

shield_status shield_kv_extend(shield_ctx *ctx, int64_t kv, const int64_t *seqs, const int32_t *counts, int32_t n) {
    return guarded([&] {
        kv::Cache &c = kv::cache_of(ctx, kv);
        kv::need(n, seqs, "seqs");
        kv::need(n, counts, "counts");
        c.book.extend(seqs, counts, n);
    });
}

shield_status shield_kv_fork(shield_ctx *ctx, int64_t kv, const int64_t *seqs, const int32_t *lens, int32_t n,
                             int64_t *out, void *stream) {
    return guarded([&] { kv::fork(ctx, kv, seqs, lens, n, out, true, stream); });
}

shield_status shield_kv_copy(shield_ctx *ctx, int64_t kv, const int64_t *seqs, const int32_t *lens, int32_t n,
                             int64_t *out, void *stream) {
    return guarded([&] { kv::fork(ctx, kv, seqs, lens, n, out, false, stream); });
}

shield_status shield_kv_free(shield_ctx *ctx, int64_t kv, const int64_t *seqs, int32_t n) {
    return guarded([&] {
        kv::Cache &c = kv::cache_of(ctx, kv);
        kv::need(n, seqs, "seqs");
        c.book.free(seqs, n);
    });
}

shield_status shield_kv_compact(shield_ctx *ctx, int64_t kv, int32_t *moved, void *stream) {
    return guarded([&] {
        kv::Cache &c = kv::cache_of(ctx, kv);
        DeviceScope scope(c.dev.ordinal);
        const cudaStream_t s = kv::stream_of(c, stream);
        kv::not_captured(s, "compacting");
        std::vector<kv::Move> moves;
        c.book.plan_compact(moves);
        kv::check(kv::launch_move_pages(c.pool, moves.data(), (int64_t)moves.size(), s), "moving pages");
        c.book.take_moves(moves);  // only now: sequences keep their pages if a launch fails
        if (moved) *moved = (int32_t)moves.size();
    });
}

shield_status shield_kv_pages(shield_ctx *ctx, int64_t kv, const int64_t *seqs, int32_t n, int32_t *lengths,
                              int32_t *pages, int32_t max_pages) {
    return guarded([&] {
        kv::Cache &c = kv::cache_of(ctx, kv);
        kv::need(n, seqs, "seqs");
        if (pages && max_pages < 0) throw Error(SHIELD_ERR_ARG, "negative count");
        for (int32_t i = 0; i < n; i++) {
            const kv::Sequence &s = c.book.get(seqs[i]);
            if (pages && (int64_t)s.pages.size() > max_pages)
                throw Error(SHIELD_ERR_RANGE, "sequence " + std::to_string(seqs[i]) + " has " +
                                                  std::to_string(s.pages.size()) + " pages, more than " + std::to_string(max_pages));
        }
        for (int32_t i = 0; i < n; i++) {
            const kv::Sequence &s = c.book.get(seqs[i]);
            if (lengths) lengths[i] = s.len;
            if (!pages) continue;
            int32_t *row = pages + (int64_t)i * max_pages;
            std::copy(s.pages.begin(), s.pages.end(), row);
            std::fill(row + s.pages.size(), row + max_pages, -1);
        }
    });
}

shield_status shield_kv_batch_create(shield_ctx *ctx, int64_t kv, const shield_kv_batch_config *cfg, int64_t *batch) {
    return guarded([&] { kv::batch_create(ctx, kv, cfg, batch); });
}

shield_status shield_kv_batch_release(shield_ctx *ctx, int64_t batch) {
    return guarded([&] {
        kv::batch_of(ctx, batch);
        kv_state(ctx).batches.erase(batch);
    });
}

shield_status shield_kv_batch_set(shield_ctx *ctx, int64_t batch, const int64_t *seqs, const int32_t *counts, int32_t n,
                                  void *stream) {
    return guarded([&] { kv::batch_set(ctx, batch, seqs, counts, n, stream); });
}

shield_status shield_kv_batch_check(shield_ctx *ctx, int64_t batch) {
    return guarded([&] { kv::check_error(kv::batch_of(ctx, batch)); });
}

shield_status shield_debug_kv_error(shield_ctx *ctx, int64_t kv, int64_t batch, int32_t word) {
    return guarded([&] {
        kv::Cache &c = kv::cache_of(ctx, kv);
        kv::Batch *B = batch ? &kv::batch_of(ctx, batch) : c.model.get();
        if (!B || B->cache != &c) throw Error(SHIELD_ERR_ARG, "the cache has no such batch");
        *static_cast<volatile int32_t *>(B->err) = word;
    });
}

shield_status shield_kv_write(shield_ctx *ctx, int64_t batch, int32_t layer, uint32_t type, const void *k,
                              int64_t k_stride, const void *v, int64_t v_stride, void *stream) {
    return guarded([&] {
        kv::Batch &B = kv::batch_of(ctx, batch);
        kv::write_rows(B, layer, type, k, k_stride, v, v_stride, kv::stream_of(*B.cache, stream));
    });
}

shield_status shield_kv_attend(shield_ctx *ctx, int64_t batch, int32_t layer, const void *q, int64_t q_stride, void *out,
                               int64_t out_stride, float scale, void *stream) {
    return guarded([&] {
        kv::Batch &B = kv::batch_of(ctx, batch);
        kv::attend(B, layer, q, q_stride, out, out_stride, scale, kv::stream_of(*B.cache, stream));
    });
}

}  // extern "C"
