// Bookkeeping of a paged key/value cache and the work plan of its attention.
// Host only (no CUDA), so it is tested without a GPU.
//
// A pool has n_pages pages of page_tokens positions. A sequence is a length
// and a list of pages: position p is row p % page_tokens of page
// list[p / page_tokens]. Pages are counted: a fork shares its parent's full
// pages. Only a sequence's last page can be partly filled, and that page is
// never shared (a fork gets a copy of it), so appending never has to copy.
#pragma once

#include <stdint.h>

#include <algorithm>
#include <deque>
#include <numeric>
#include <string>
#include <unordered_map>
#include <unordered_set>
#include <vector>

#include "error.h"

namespace shield {
namespace kv {

// Rows [0, rows) of page src, in every layer and head, become those of page dst.
struct Move {
    int32_t src, dst, rows;
};

struct Sequence {
    int32_t len = 0;
    std::vector<int32_t> pages;
};

class Pool {
public:
    // `number` tells this pool's sequences from other pools': it is the upper
    // bits of their ids.
    Pool(int32_t n_pages, int32_t page_tokens, int64_t number)
        : page_tokens_(page_tokens), free_count_(n_pages), number_(number), ref_(n_pages, 0),
          free_((size_t)(n_pages + 63) / 64, 0) {
        for (int32_t p = 0; p < n_pages; p++) free_[p >> 6] |= uint64_t(1) << (p & 63);
    }

    int32_t page_tokens() const { return page_tokens_; }
    int32_t n_pages() const { return (int32_t)ref_.size(); }
    int32_t pages_used() const { return n_pages() - free_count_; }
    int32_t sequences() const { return (int32_t)(slots_.size() - idle_.size()) - spent_; }
    // One past the highest page in use.
    int32_t pages_spanned() const {
        int32_t p = n_pages();
        while (p > 0 && ref_[p - 1] == 0) p--;
        return p;
    }
    // Counts the calls that took pages away from a sequence or moved them:
    // plans made before may point at the wrong rows.
    int64_t frees() const { return frees_; }
    int64_t moves() const { return moves_; }

    const Sequence &get(int64_t id) const { return slot(id).s; }
    bool has(int64_t id) const { return find(id) != nullptr; }
    int32_t holders(int32_t page) const { return ref_[page]; }

    void open(int32_t n, int64_t *out) {
        room(n);
        for (int32_t i = 0; i < n; i++) out[i] = begin();
    }

    // Adds count[i] positions to sequence ids[i]; all of them or none.
    void extend(const int64_t *ids, const int32_t *count, int32_t n) {
        distinct(ids, n);
        int64_t need = 0;
        for (int32_t i = 0; i < n; i++) {
            const Sequence &s = get(ids[i]);
            if (count[i] < 0) throw Error(SHIELD_ERR_RANGE, "sequence " + std::to_string(ids[i]) + ": negative count");
            const int64_t len = (int64_t)s.len + count[i];
            if (len > INT32_MAX - 256) throw Error(SHIELD_ERR_RANGE, "sequence " + std::to_string(ids[i]) + " would be too long");
            need += pages_of(len) - (int64_t)s.pages.size();
        }
        reserve(need);
        for (int32_t i = 0; i < n; i++) {
            Sequence &s = slot(ids[i]).s;
            s.len += count[i];
            while ((int64_t)s.pages.size() < pages_of(s.len)) s.pages.push_back(take());
        }
    }

    // Takes back what the latest extend() of these sequences added. (Plans made
    // before it still hold.)
    void undo_extend(const int64_t *ids, const int32_t *count, int32_t n) {
        for (int32_t i = 0; i < n; i++) {
            Sequence &s = slot(ids[i]).s;
            s.len -= count[i];
            while ((int64_t)s.pages.size() > pages_of(s.len)) {
                const int32_t p = s.pages.back();
                s.pages.pop_back();
                if (--ref_[p] == 0) give(p);
            }
        }
    }

    // Child i: the first len[i] positions (null: all) of parents[i], sharing
    // its full pages (share) or with a copy of every page.
    void fork(const int64_t *parents, const int32_t *len, int32_t n, bool share, int64_t *out, std::vector<Move> &moves) {
        int64_t need = 0;
        for (int32_t i = 0; i < n; i++) {
            const Sequence &s = get(parents[i]);
            const int32_t l = len ? len[i] : s.len;
            if (l < 0 || l > s.len)
                throw Error(SHIELD_ERR_RANGE, "sequence " + std::to_string(parents[i]) + " holds " +
                                                  std::to_string(s.len) + " positions, not " + std::to_string(l));
            need += share ? (l % page_tokens_ != 0) : pages_of(l);
        }
        reserve(need);
        room(n);
        moves.reserve((size_t)need);
        for (int32_t i = 0; i < n; i++) {
            const int64_t child = begin();
            const Sequence &s = slot(parents[i]).s;  // (slots stay where they are)
            Sequence &c = slot(child).s;
            out[i] = child;
            c.len = len ? len[i] : s.len;
            c.pages.reserve((size_t)pages_of(c.len) + 1);
            for (int32_t j = 0; j < pages_of(c.len); j++) {
                const int32_t rows = std::min(page_tokens_, c.len - j * page_tokens_);
                if (share && rows == page_tokens_) {
                    ref_[s.pages[j]]++;
                    c.pages.push_back(s.pages[j]);
                } else {
                    const int32_t p = take();
                    moves.push_back({s.pages[j], p, rows});
                    c.pages.push_back(p);
                }
            }
        }
    }

    void free(const int64_t *ids, int32_t n) {
        distinct(ids, n);
        for (int32_t i = 0; i < n; i++) get(ids[i]);
        for (int32_t i = 0; i < n; i++) {
            Slot &t = slot(ids[i]);
            for (int32_t p : t.s.pages)
                if (--ref_[p] == 0) give(p);
            t.s.pages.clear();  // keeps its memory for the slot's next sequence
            t.s.len = 0;
            t.live = false;
            if (++t.turn <= TURN_MASK) idle_.push_back((int32_t)(ids[i] & SLOT_MASK));
            else spent_++;  // its ids are used up: one that ended long ago must not name another sequence
        }
        if (n > 0) frees_++;
    }

    // The i-th highest used page moves to the i-th lowest free one while that
    // is lower; afterwards the used pages are the lowest ones. The pages read
    // and the pages written are disjoint, so the moves may run in any order.
    // Nothing changes before take_moves(), when the rows are on their way: until
    // then what was copied lies in free pages.
    void plan_compact(std::vector<Move> &moves) const {
        std::vector<int32_t> to((size_t)n_pages(), -1);
        int32_t lo = 0, hi = n_pages() - 1;
        for (;;) {
            while (lo < hi && ref_[lo] != 0) lo++;
            while (hi > lo && ref_[hi] == 0) hi--;
            if (lo >= hi) break;
            to[hi] = (int32_t)moves.size();
            moves.push_back({hi, lo, 0});
            lo++;
            hi--;
        }
        if (moves.empty()) return;
        for (const Slot &t : slots_) {
            const Sequence &s = t.s;  // (an idle slot has no pages)
            for (int32_t j = 0; j < (int32_t)s.pages.size(); j++) {
                const int32_t m = to[s.pages[j]];
                if (m >= 0) moves[m].rows = std::max(moves[m].rows, std::min(page_tokens_, s.len - j * page_tokens_));
            }
        }
    }
    // What plan_compact() gave, with no other call in between.
    void take_moves(const std::vector<Move> &moves) {
        if (moves.empty()) return;
        std::vector<int32_t> to((size_t)n_pages());
        std::iota(to.begin(), to.end(), 0);
        for (const Move &m : moves) to[m.src] = m.dst;
        for (Slot &t : slots_)
            for (int32_t &p : t.s.pages) p = to[p];
        for (const Move &m : moves) {
            std::swap(ref_[m.src], ref_[m.dst]);
            free_[m.dst >> 6] &= ~(uint64_t(1) << (m.dst & 63));
            free_[m.src >> 6] |= uint64_t(1) << (m.src & 63);
        }
        hint_ = 0;
        moves_++;
    }
    void compact(std::vector<Move> &moves) {
        plan_compact(moves);
        take_moves(moves);
    }

private:
    int32_t pages_of(int64_t len) const { return (int32_t)((len + page_tokens_ - 1) / page_tokens_); }
    void reserve(int64_t need) const {
        if (need > free_count_)
            throw Error(SHIELD_ERR_NOMEM, "the call needs " + std::to_string(need) + " pages; the pool has " +
                                              std::to_string(free_count_) + " free");
    }
    int32_t take() {  // the lowest free page; reserve() came first
        while (!free_[hint_]) hint_++;
        const int32_t p = (int32_t)(hint_ * 64 + (size_t)__builtin_ctzll(free_[hint_]));
        free_[hint_] &= free_[hint_] - 1;
        ref_[p] = 1;
        free_count_--;
        return p;
    }
    void give(int32_t p) {
        free_[p >> 6] |= uint64_t(1) << (p & 63);
        hint_ = std::min(hint_, (size_t)(p >> 6));
        free_count_++;
    }
    void distinct(const int64_t *ids, int32_t n) const {
        if (n < 2) return;
        call_++;
        for (int32_t i = 0; i < n; i++) {
            const Slot &t = slot(ids[i]);
            if (t.call == call_)
                throw Error(SHIELD_ERR_ARG, "sequence " + std::to_string(ids[i]) + " appears twice in one call");
            t.call = call_;
        }
    }

    // An id is the pool's number, the turn of its slot (how many sequences that
    // had before) and the slot.
    static constexpr int SLOT_BITS = 22, TURN_BITS = 22;
    static constexpr int64_t SLOT_MASK = (1 << SLOT_BITS) - 1, TURN_MASK = (1 << TURN_BITS) - 1;
    struct Slot {
        Sequence s;
        int64_t turn = 0;
        bool live = false;
        mutable uint64_t call = 0;  // the last call that named it (distinct)
    };
    const Slot *find(int64_t id) const {
        const int64_t at = id & SLOT_MASK;
        if (id >> (SLOT_BITS + TURN_BITS) != number_ || at >= (int64_t)slots_.size()) return nullptr;
        const Slot &t = slots_[(size_t)at];
        return t.live && t.turn == ((id >> SLOT_BITS) & TURN_MASK) ? &t : nullptr;
    }
    const Slot &slot(int64_t id) const {
        const Slot *t = find(id);
        if (!t) throw Error(SHIELD_ERR_ARG, "unknown sequence " + std::to_string(id) + " of this pool");
        return *t;
    }
    Slot &slot(int64_t id) { return const_cast<Slot &>(const_cast<const Pool *>(this)->slot(id)); }
    void room(int32_t n) const {
        if ((int64_t)slots_.size() - (int64_t)idle_.size() + n > SLOT_MASK + 1)
            throw Error(SHIELD_ERR_NOMEM, "more sequences than a pool takes");
    }
    int64_t begin() {  // an empty sequence; room() came first
        int64_t at;
        if (idle_.empty()) {
            at = (int64_t)slots_.size();
            slots_.emplace_back();
        } else {
            at = idle_.back();
            idle_.pop_back();
        }
        Slot &t = slots_[(size_t)at];
        t.live = true;
        return number_ << (SLOT_BITS + TURN_BITS) | t.turn << SLOT_BITS | at;
    }

    int32_t page_tokens_, free_count_;
    int64_t number_, frees_ = 0, moves_ = 0;
    mutable uint64_t call_ = 0;
    std::vector<int32_t> ref_;     // sequences holding each page
    std::vector<uint64_t> free_;   // one bit per page
    size_t hint_ = 0;              // no free page in a word before this one
    std::deque<Slot> slots_;
    std::vector<int32_t> idle_;    // slots without a sequence
    int32_t spent_ = 0;            // slots that take no sequence any more
};

// Whether two sequences have a page in common among those of their last count[i]
// positions. (It is full, and the last positions of each reach its end.)
inline bool steps_meet(const Pool &pool, const int64_t *ids, const int32_t *count, int32_t n) {
    std::unordered_set<int32_t> seen;
    for (int32_t i = 0; i < n; i++) {
        const Sequence &s = pool.get(ids[i]);
        if (count[i] <= 0) continue;
        for (size_t j = (size_t)((s.len - count[i]) / pool.page_tokens()); j < s.pages.size(); j++)
            if (pool.holders(s.pages[j]) > 1 && !seen.insert(s.pages[j]).second) return true;
    }
    return false;
}

// The capacity to make for `need` where there is room for `have`: a power of
// two up to `most`, so that a sequence that grows by a token a step outgrows it
// a few times in all.
inline int32_t grown(int32_t have, int32_t need, int32_t most) {
    if (need <= have) return have;
    int64_t c = 1;
    while (c < need) c *= 2;
    return (int32_t)std::max<int64_t>(need, std::min<int64_t>(c, most));
}

// ------------------------------------------------------------- attention plan

// One piece of attention work for every kv head: rows [r0, r0 + nr) of a
// segment against keys [k0, k1). A segment's rows are its tokens times the
// query heads of a kv head: row r is token perm[tok0 + r / G], head r % G.
struct Item {
    int32_t tok0, r0, nr;
    int32_t k0, k1;
    int32_t table;   // where the page list of position 0 starts in the table
    int32_t part;    // first partial row (kv head j's rows follow at part + j * nr), or -1: rows go straight out
    int32_t masked;  // some row stops before k1
};

// Keys that a set of tokens attends to together: a run of pages that several
// sequences share, or (a leaf) the rest of one sequence. Its rows (tokens times
// query heads of a kv head) are cut into ntiles tiles of tile_rows, its keys
// into nsplit pieces; the item of piece s and tile t has its partial rows from
// where[slot0 + s * ntiles + t] on (-1: it has none).
struct Segment {
    int32_t tok0, rows, slot0, ntiles, nsplit, tile_rows, parent, direct;
};
// A token whose rows are joined from partials: its place in plan order, its
// batch token and its leaf segment.
struct Join {
    int32_t at, token, leaf;
};

struct PlanShape {
    int32_t group = 1;         // query heads per kv head
    int32_t kv_heads = 1;
    int32_t sms = 148;
    int32_t few_rows = 16;     // segments up to this many rows take the few-row kernel
    int64_t max_items = 0;     // capacity: items of either kind
    int64_t max_segments = 0;  // capacity: segments
    int64_t max_part = 0;      // capacity: partial rows
    int64_t max_table = 0;     // capacity: page table entries
};

struct Plan {
    std::vector<int32_t> slot;             // per batch token: page * page_tokens + row, where its key and value go
    std::vector<int32_t> perm, lim;        // per token in plan order: batch token, visible keys
    std::vector<Segment> segs;
    std::vector<Item> few, tile;           // longest first
    std::vector<int32_t> where;            // first partial row of each segment slot, -1: none
    std::vector<Join> merge;
    std::vector<int32_t> table;
    int64_t part_rows = 0;
    int32_t solo = 0;                      // the last items of few, which a warp takes alone
    void clear() {
        slot.clear(); perm.clear(); lim.clear(); segs.clear(); few.clear(); tile.clear(); where.clear(); merge.clear();
        table.clear();
        part_rows = 0;
        solo = 0;
    }
};

constexpr int32_t FEW_TILE = 16;  // rows of a few-row item
constexpr int32_t FEW_SOLO = 64;  // keys that one warp may take alone
constexpr int32_t KEY_STEP = 128; // splits are whole steps of this many keys

namespace detail {

struct Draft {  // a segment before its items are made
    int32_t tok0, ntok, k0, k1, table, parent;
    bool leaf;
};

}  // namespace detail

// Plans the attention of the last count[i] positions of each sequence over
// their histories. Sequences whose page lists begin alike form a tree; a run
// of pages common to several of them becomes one segment for all their tokens
// where that is worth it (share), and long segments are cut along the keys
// (split). False: the plan does not fit the capacities.
inline bool make_plan_with(const Pool &pool, const int64_t *ids, const int32_t *count, int32_t n, const PlanShape &S,
                           bool share, bool split, Plan &P) {
    using detail::Draft;
    P.clear();
    const int32_t pt = pool.page_tokens(), G = S.group;
    struct Member {
        const Sequence *s;
        int32_t count, tok, shared, table;  // shared: pages that end before its new tokens
    };
    std::vector<Member> mem;
    int32_t tok = 0;
    for (int32_t i = 0; i < n; i++) {
        const Sequence &s = pool.get(ids[i]);
        if (count[i] > 0) {
            const int32_t used = (s.len + pt - 1) / pt;
            mem.push_back({&s, count[i], tok, (s.len - count[i]) / pt, (int32_t)P.table.size()});
            if ((int64_t)P.table.size() + used > S.max_table) return false;
            P.table.insert(P.table.end(), s.pages.begin(), s.pages.begin() + used);
            for (int32_t p = s.len - count[i]; p < s.len; p++) P.slot.push_back(s.pages[p / pt] * pt + p % pt);
        }
        tok += count[i];
    }
    // The tree, depth first, so that every node's tokens are neighbours.
    struct Node {
        std::vector<int32_t> members;
        int32_t start, at, parent;  // first page not yet attended to, page to split by
    };
    std::vector<Node> stack;
    std::vector<Draft> drafts;
    std::vector<int32_t> leaf;  // of each token in plan order
    {
        Node root{{}, 0, 0, -1};
        for (int32_t i = 0; i < (int32_t)mem.size(); i++) root.members.push_back(i);
        if (!mem.empty()) stack.push_back(std::move(root));
    }
    while (!stack.empty()) {
        Node nd = std::move(stack.back());
        stack.pop_back();
        std::vector<std::vector<int32_t>> groups;  // by the page at nd.at, in order of appearance
        std::unordered_map<int32_t, size_t> by_page;
        for (int32_t m : nd.members) {
            if (!share || mem[m].shared <= nd.at) {
                groups.push_back({m});
                continue;
            }
            auto r = by_page.emplace(mem[m].s->pages[nd.at], groups.size());
            if (r.second) groups.push_back({m});
            else groups[r.first->second].push_back(m);
        }
        if (groups.size() > 1) {
            for (size_t g = groups.size(); g-- > 0;)
                stack.push_back({std::move(groups[g]), nd.start, nd.at, nd.parent});
            continue;  // each comes back as the only group of its node
        }
        const std::vector<int32_t> &g = groups[0];
        const Member &first = mem[g[0]];
        if (g.size() == 1) {
            const int32_t t0 = (int32_t)P.perm.size(), len = first.s->len;
            for (int32_t j = 0; j < first.count; j++) {
                P.perm.push_back(first.tok + j);
                P.lim.push_back(len - first.count + j + 1);
                leaf.push_back((int32_t)drafts.size());
            }
            drafts.push_back({t0, first.count, nd.start * pt, len, first.table, nd.parent, true});
            continue;
        }
        int32_t end = first.shared;
        for (size_t i = 1; i < g.size(); i++) {
            const Member &m = mem[g[i]];
            end = std::min(end, m.shared);
            int32_t c = nd.at;
            while (c < end && m.s->pages[c] == first.s->pages[c]) c++;
            end = c;
        }
        // Sharing pays when the separate passes over these keys cost more than
        // one pass for all rows plus the partial results of every row (two
        // per row, written and read back). In SM cycles per 128 keys: a pass
        // of up to 128 rows is bound by loading keys and values (about 1400),
        // 256 rows by their products (about 2048); a row's partials about 90.
        auto pass = [](int64_t rows) -> int64_t { return rows <= 128 ? 1400 : (rows + 255) / 256 * 2048; };
        int64_t apart = 0, rows = 0;
        for (int32_t m : g) {
            apart += pass((int64_t)mem[m].count * G);
            rows += (int64_t)mem[m].count * G;
        }
        const int64_t keys = (int64_t)(end - nd.start) * pt;
        const bool pays = (apart - pass(rows)) * keys > 90 * rows * KEY_STEP;
        Node next{g, nd.start, end, nd.parent};
        if (pays) {
            int32_t ntok = 0;
            for (int32_t m : g) ntok += mem[m].count;
            next.parent = (int32_t)drafts.size();
            next.start = end;
            drafts.push_back({(int32_t)P.perm.size(), ntok, nd.start * pt, end * pt, first.table, nd.parent, false});
        }
        stack.push_back(std::move(next));
    }
    auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    auto is_few = [&](const Draft &d) { return (int64_t)d.ntok * G <= S.few_rows; };
    auto steps_of = [&](const Draft &d) { return up(d.k1 - d.k0, KEY_STEP); };
    int64_t wide_units = 0;
    for (const Draft &d : drafts)
        if (!is_few(d)) wide_units += up((int64_t)d.ntok * G, 256);
    // 256-row tiles share each key block between two row blocks; 128-row ones
    // when 256-row ones would leave SMs idle
    const int32_t wide = wide_units * S.kv_heads < S.sms ? 128 : 256;
    auto tile_rows = [&](const Draft &d) {
        if (is_few(d)) return FEW_TILE;
        return (int64_t)d.ntok * G <= 128 ? 128 : wide;
    };
    // How many steps of keys a piece may have: of the lengths tried, the one with
    // the least estimated time on `slots` places that work side by side. Up to a
    // few rounds of pieces the rounds count, each as long as a longest piece and
    // `extra` steps for its start and end; beyond that the sum.
    auto piece_steps = [&](bool few, int64_t slots, int64_t extra, int64_t least) {
        int64_t longest = 0;
        for (const Draft &d : drafts)
            if (is_few(d) == few) longest = std::max(longest, steps_of(d));
        if (longest <= least || !split) return std::max<int64_t>(longest, 1);
        int64_t best = longest;
        double best_time = 1e300;
        for (int64_t n = 1; n <= std::min<int64_t>(longest / least + 1, 64); n++) {
            const int64_t c = std::max(least, up(longest, n));
            int64_t units = 0, work = 0;
            for (const Draft &d : drafts)
                if (is_few(d) == few) {
                    const int64_t tiles = up((int64_t)d.ntok * G, tile_rows(d)), pieces = up(steps_of(d), c);
                    units += tiles * pieces * S.kv_heads;
                    work += tiles * S.kv_heads * (steps_of(d) + pieces * extra);
                }
            const double sum = (double)work / (double)slots + 0.5 * (double)(c + extra);
            const double rounds = (double)up(units, slots) * (double)(c + extra);
            const double time = std::max((double)(c + extra), units <= 4 * slots ? std::min(rounds, 2 * sum) : sum) + (n > 1 ? 1.0 : 0.0);
            if (time < best_time - 1e-9) {
                best_time = time;
                best = c;
            }
        }
        return best;
    };
    const int64_t few_chunk = piece_steps(true, (int64_t)S.sms * 2, 3, 4) * KEY_STEP;
    const int64_t tile_chunk = piece_steps(false, S.sms, 4, 4) * KEY_STEP;
    struct Ref {
        int64_t cost;
        Item it;
        bool few;
    };
    std::vector<Ref> refs;
    for (const Draft &d : drafts) {
        Segment sg;
        const int64_t rows = (int64_t)d.ntok * G, keys = d.k1 - d.k0;
        const bool few = is_few(d);
        sg.tok0 = d.tok0;
        sg.rows = (int32_t)rows;
        sg.slot0 = (int32_t)P.where.size();
        sg.tile_rows = tile_rows(d);
        sg.ntiles = (int32_t)up(rows, sg.tile_rows);
        sg.nsplit = split ? (int32_t)up(keys, few ? few_chunk : tile_chunk) : 1;
        sg.parent = d.parent;
        sg.direct = d.leaf && d.parent < 0 && sg.nsplit == 1;
        const int64_t step = up(up(keys, sg.nsplit), KEY_STEP) * KEY_STEP;
        if ((int64_t)P.where.size() + (int64_t)sg.nsplit * sg.ntiles > S.max_items) return false;
        for (int32_t sp = 0; sp < sg.nsplit; sp++)
            for (int32_t t = 0; t < sg.ntiles; t++) {
                Item it;
                it.tok0 = d.tok0;
                it.r0 = t * sg.tile_rows;
                it.nr = (int32_t)std::min<int64_t>(sg.tile_rows, rows - it.r0);
                it.k0 = (int32_t)std::min<int64_t>(d.k1, d.k0 + sp * step);
                it.k1 = (int32_t)std::min<int64_t>(d.k1, d.k0 + (sp + 1) * step);
                it.table = d.table;
                it.part = -1;
                it.masked = 0;
                if (d.leaf) {
                    it.k1 = std::min(it.k1, P.lim[d.tok0 + (it.r0 + it.nr - 1) / G]);
                    it.masked = P.lim[d.tok0 + it.r0 / G] < it.k1;
                }
                if (it.k1 <= it.k0) {  // causal: no key of this piece is visible
                    P.where.push_back(-1);
                    continue;
                }
                if (!sg.direct) {
                    it.part = (int32_t)P.part_rows;
                    P.part_rows += (int64_t)it.nr * S.kv_heads;
                    if (P.part_rows > S.max_part) return false;
                }
                const int64_t cost = (int64_t)(it.k1 - it.k0) * (it.nr > 128 ? 2 : 1);
                refs.push_back({cost, it, few});
                P.where.push_back(it.part);
            }
        P.segs.push_back(sg);
    }
    if ((int64_t)P.segs.size() > S.max_segments) return false;
    std::stable_sort(refs.begin(), refs.end(), [](const Ref &a, const Ref &b) { return a.cost > b.cost; });
    for (const Ref &r : refs) (r.few ? P.few : P.tile).push_back(r.it);
    // short pieces go to single warps when there are more than CTAs side by side
    if ((int64_t)P.few.size() * S.kv_heads > 2 * (int64_t)S.sms)
        for (const Item &it : P.few) P.solo += it.k1 - it.k0 <= FEW_SOLO;
    for (int32_t t = 0; t < (int32_t)P.perm.size(); t++)
        if (!P.segs[leaf[t]].direct) P.merge.push_back({t, P.perm[t], leaf[t]});
    return true;
}

// The plan with the most sharing and splitting that fits the capacities; the
// last one tried needs one item per row tile and no partial rows.
inline void make_plan(const Pool &pool, const int64_t *ids, const int32_t *count, int32_t n, const PlanShape &S, Plan &P) {
    if (make_plan_with(pool, ids, count, n, S, true, true, P)) return;
    if (make_plan_with(pool, ids, count, n, S, true, false, P)) return;
    if (make_plan_with(pool, ids, count, n, S, false, false, P)) return;
    throw Error(SHIELD_ERR_RANGE, "the plan exceeds the batch's capacities");
}

}  // namespace kv
}  // namespace shield
