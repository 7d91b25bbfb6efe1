// C entry points to the cache's host bookkeeping, for tests without a GPU.
#include <cstring>

#include "kv_pool.h"

using namespace shield;
using namespace shield::kv;

struct Host {
    Pool pool;
    Plan plan;
    std::vector<Move> moves;
    std::string error;
    int32_t code = 0;
};

template <class F>
static int32_t run(Host *h, F &&f) {
    try {
        f();
        h->error.clear();
        return h->code = SHIELD_OK;
    } catch (const Error &e) {
        h->error = e.what();
        return h->code = e.code;
    }
}

extern "C" {

Host *host_new(int32_t pages, int32_t page_tokens) { return new Host{Pool(pages, page_tokens, 1), {}, {}, "", 0}; }
void host_delete(Host *h) { delete h; }
const char *host_error(Host *h) { return h->error.c_str(); }
int32_t host_open(Host *h, int32_t n, int64_t *out) { return run(h, [&] { h->pool.open(n, out); }); }
int32_t host_extend(Host *h, const int64_t *ids, const int32_t *c, int32_t n) { return run(h, [&] { h->pool.extend(ids, c, n); }); }
int32_t host_fork(Host *h, const int64_t *ids, const int32_t *len, int32_t n, int32_t share, int64_t *out) {
    return run(h, [&] { h->moves.clear(); h->pool.fork(ids, len, n, share != 0, out, h->moves); });
}
int32_t host_free(Host *h, const int64_t *ids, int32_t n) { return run(h, [&] { h->pool.free(ids, n); }); }
int32_t host_compact(Host *h) { return run(h, [&] { h->moves.clear(); h->pool.compact(h->moves); }); }
int32_t host_plan_compact(Host *h) { return run(h, [&] { h->moves.clear(); h->pool.plan_compact(h->moves); }); }
int32_t host_moves(Host *h, int32_t *out) {
    if (out && !h->moves.empty()) memcpy(out, h->moves.data(), h->moves.size() * sizeof(Move));
    return (int32_t)h->moves.size();
}
int32_t host_used(Host *h) { return h->pool.pages_used(); }
int32_t host_spanned(Host *h) { return h->pool.pages_spanned(); }
int32_t host_len(Host *h, int64_t id) { return h->pool.get(id).len; }
int32_t host_pages(Host *h, int64_t id, int32_t *out) {
    const Sequence &s = h->pool.get(id);
    if (out) std::copy(s.pages.begin(), s.pages.end(), out);
    return (int32_t)s.pages.size();
}
// few_rows, capacities as in PlanShape; mode: 0 make_plan, 1..3 its three tries alone
int32_t host_plan(Host *h, const int64_t *ids, const int32_t *c, int32_t n, int32_t group, int32_t kv_heads, int32_t few_rows,
                  int64_t max_items, int64_t max_segments, int64_t max_part, int64_t max_table, int32_t mode) {
    PlanShape S;
    S.group = group;
    S.kv_heads = kv_heads;
    S.few_rows = few_rows;
    S.max_items = max_items;
    S.max_segments = max_segments;
    S.max_part = max_part;
    S.max_table = max_table;
    int32_t fits = 1;
    const int32_t rc = run(h, [&] {
        if (mode == 0) make_plan(h->pool, ids, c, n, S, h->plan);
        else fits = make_plan_with(h->pool, ids, c, n, S, mode < 3, mode < 2, h->plan);
    });
    return rc ? rc : fits ? 0 : -1;
}
// which: 0 slot, 1 perm, 2 lim, 3 merge, 4 segs, 5 few, 6 tile, 7 where, 8 table; returns int32 words
int64_t host_plan_array(Host *h, int32_t which, int32_t *out) {
    const Plan &P = h->plan;
    auto give = [&](const void *p, size_t words) {
        if (out && words) memcpy(out, p, words * 4);
        return (int64_t)words;
    };
    switch (which) {
    case 0: return give(P.slot.data(), P.slot.size());
    case 1: return give(P.perm.data(), P.perm.size());
    case 2: return give(P.lim.data(), P.lim.size());
    case 3: return give(P.merge.data(), P.merge.size() * sizeof(Join) / 4);
    case 4: return give(P.segs.data(), P.segs.size() * sizeof(Segment) / 4);
    case 5: return give(P.few.data(), P.few.size() * sizeof(Item) / 4);
    case 6: return give(P.tile.data(), P.tile.size() * sizeof(Item) / 4);
    case 7: return give(P.where.data(), P.where.size());
    case 8: return give(P.table.data(), P.table.size());
    }
    return -1;
}
int32_t host_grown(int32_t have, int32_t need, int32_t most) { return grown(have, need, most); }
int32_t host_steps_meet(Host *h, const int64_t *ids, const int32_t *c, int32_t n) { return steps_meet(h->pool, ids, c, n); }
// n sequences opened and freed one after another: how many had the id of the first or of the one before
int64_t host_churn(Host *h, int64_t n) {
    int64_t first = 0, last = 0, id = 0, again = 0;
    for (int64_t i = 0; i < n; i++) {
        h->pool.open(1, &id);
        if (i == 0) first = id;
        else again += id == first || id == last;
        last = id;
        h->pool.free(&id, 1);
    }
    return again;
}
int32_t host_sequences(Host *h) { return h->pool.sequences(); }
int64_t host_part_rows(Host *h) { return h->plan.part_rows; }

}  // extern "C"
