// Host plan of one step's attention over the paged cache: which rows read
// which keys, in pieces that fill the GPU.  Plain C++ with no device code.
//
// A row is one query head of one token; the G query heads that share a kv
// head make G consecutive rows of a token, and everything below is per kv
// head (the kernel's grid has the kv heads as its second factor).
//
// Sequences are sorted by their page lists, so that those with a common start
// lie side by side, and walked as a tree: a run of whole pages that several
// sequences share, all of it before each one's first new token, becomes one
// segment with the rows of all of them, when the bytes this saves outweigh
// the partial results it adds; what is left of a sequence is a segment of its
// own with the causal limit.  A segment's rows are cut into tiles and its keys
// into pieces of about equal length.  Rows whose keys lie in several pieces
// get a partial result from each and are joined by a second kernel.
#pragma once

#include <algorithm>
#include <cstdint>
#include <functional>
#include <vector>

#include "kv_tables.h"

namespace exq {

// One workgroup's work for one kv head: rows [row0, row0 + n_rows) of the
// plan's row order against the keys at positions [key0, key1), the page of
// position p being pages[page_at + p / page_tokens] (an index into the plan's
// words).  causal: a row sees positions up to its token's own only.  part: the
// partial result of row row0 (rows follow), -1 when the rows have no other
// piece and the result is final.
struct AttnItem {
    int32_t row0, n_rows, key0, key1, page_at, causal, part, pad;
};
// One token: its place in the sequence and its slot in the pool (page *
// page_tokens + offset), and, for plan order: the token that stands there and
// that one's position.
struct PlanToken {
    int32_t pos, slot, order, order_pos;
};
struct PlanHeader {
    int32_t n_tokens, n_items, n_joined;  // n_joined: rows with more than one piece
    int32_t join_rows;                    // word index of the joined rows' numbers
    int32_t join_at;                      // n_joined + 1 word indices into the partial numbers
    int32_t parts;                        // partial results of one kv head
    int32_t pad[10];
};
static_assert(sizeof(AttnItem) == 32 && sizeof(PlanToken) == 16 && sizeof(PlanHeader) == 64, "words of the device plan");

// What a workgroup takes for one key, in tenths of a nanosecond with all others
// at work, for at most 16, 32, 64 and 128 rows (0: not that many at once).
struct RowCost {
    int of[4];
};
// Of csrc/attn.hip's kernel for a cache of f32 (type 0), f16 (1) or Q8_0 (8) and
// heads of 64, 96, 128 or 256.  0: it has no form for as many (Geo::ONE, RT).
// Measured: 8 kv heads, 512 workgroups at once (f32 and f16 at 256: 256); keys of
// 4096 tokens a sequence for few rows (bound by the loads, 5 to 6 TB/s), of one run
// of 131072 for more, which no L2 holds: a chunk behind 8192 keys takes two thirds.
inline RowCost attn_cost(int type, int dim) {
    const int d = dim == 64 ? 0 : dim == 96 ? 1 : dim == 128 ? 2 : 3;
    static const RowCost f32[4] = {{{460, 540, 1000, 1580}}, {{666, 797, 1494, 2270}}, {{878, 1007, 1780, 2900}}, {{867, 2120, 2122, 0}}};
    static const RowCost f16[4] = {{{237, 320, 320, 520}}, {{336, 470, 480, 730}}, {{474, 590, 595, 840}}, {{433, 648, 650, 0}}};
    static const RowCost q80[4] = {{{148, 267, 0, 774}}, {{230, 403, 0, 1100}}, {{286, 469, 920, 1160}}, {{577, 0, 0, 0}}};
    return type == 0 ? f32[d] : type == 1 ? f16[d] : q80[d];
}

struct PlanShape {
    int group;       // query heads of one kv head
    int n_kv;
    RowCost cost;
    int part_cost;   // a row's partial result, written and read, in the same unit
    int workgroups;  // that run at once
    int min_cost;    // a piece of fewer keys than this takes is not worth its start (of 64 to 256 keys)
};

struct AttnPlan {
    static constexpr int kKeyStep = 64;     // pieces are multiples of it

    std::vector<PlanToken> tokens;  // by token; order fields by plan order
    std::vector<AttnItem> items;    // page_at, relative to `pages`
    std::vector<int32_t> pages;
    std::vector<int32_t> join_rows, join_at, join_parts;
    int parts = 0;
    bool writable = true;  // no new token's page has another holder

    void build(const KvTables &kv, int n, const int *seqs, const int *n_new, const PlanShape &shape) {
        kv_ = &kv;
        shape_ = shape;
        pt_ = kv.page_tokens();
        tokens.clear();
        items.clear();
        pages.clear();
        join_rows.clear();
        join_at.clear();
        join_parts.clear();
        segs_.clear();
        parts = 0;
        writable = true;
        weigh();
        nodes_.clear();
        for (int i = 0; i < n; ++i) {
            const KvTables::Seq &s = kv.seq(seqs[i]);
            const int first = (int)tokens.size(), q0 = s.len - n_new[i];
            for (int p = q0; p < s.len; ++p) {
                const int page = s.pages[(size_t)p / pt_];
                if (kv.holders(page) > 1) writable = false;
                tokens.push_back({p, page * pt_ + p % pt_, 0, 0});
            }
            if (n_new[i] > 0) nodes_.push_back({&s, first, n_new[i], q0 / pt_, 0});
        }
        if (tokens.empty()) return;
        std::stable_sort(nodes_.begin(), nodes_.end(), [](const Node &a, const Node &b) {
            const int most = std::min(a.shareable, b.shareable), d = agree(a, b, 0, most);
            return d < most ? a.seq->pages[d] < b.seq->pages[d] : a.shareable < b.shareable;
        });
        int at = 0;
        for (Node &nd : nodes_) {
            nd.row0 = at * shape_.group;
            for (int t = 0; t < nd.n_new; ++t, ++at) {
                tokens[at].order = nd.first + t;
                tokens[at].order_pos = tokens[nd.first + t].pos;
            }
        }
        walk();
        cut((int)tokens.size() * shape_.group);
    }

  private:
    struct Node {
        const KvTables::Seq *seq;
        int first, n_new, shareable, row0;  // shareable: whole pages before the first new token
    };
    struct Segment {
        int row0, n_rows, key0, key1, page_at, causal;
    };
    struct Span {
        int lo, hi, start, depth;  // nodes [lo, hi) share their first `depth` pages; pages from `start` on are unread
    };

    // How many leading pages two sequences have in common, at least `from` and at
    // most `most`.  Pages are only shared by forks, which share a whole start: a
    // page in common means that all before it are, so a binary search finds the end.
    static int agree(const Node &a, const Node &b, int from, int most) {
        while (from < most) {
            const int mid = from + (most - from) / 2;
            if (a.seq->pages[mid] == b.seq->pages[mid]) from = mid + 1;
            else most = mid;
        }
        return from;
    }

    // The cheapest cut of up to 8 units of 16 rows into workgroups of 1, 2, 4 and 8: its cost and its first piece, the
    // larger of equals.
    void weigh() {
        best_[0] = 0;
        for (int n = 1; n <= 8; ++n) {
            step_[n] = 0;
            for (int k = 3; k >= 0; --k) {
                if (shape_.cost.of[k] == 0) continue;
                const int u = 1 << k, c = shape_.cost.of[k] + best_[n > u ? n - u : 0];
                if (step_[n] == 0 || c < best_[n]) {
                    best_[n] = c;
                    step_[n] = u;
                }
            }
        }
    }
    // How many of `rows` rows the next workgroup takes.
    int tile(int rows) const { return std::min(rows, 16 * step_[std::min(8, (rows + 15) / 16)]); }
    int tile_cost(int rows) const { return shape_.cost.of[rows <= 16 ? 0 : rows <= 32 ? 1 : rows <= 64 ? 2 : 3]; }
    // Of one key for these rows.
    long long cost(int rows) const { return (long long)(rows / 128) * best_[8] + best_[(rows % 128 + 15) / 16]; }

    int list_pages(const KvTables::Seq &s, int from, int to) {
        // positions keep their own page index: pages[at + p / page_tokens]
        const int at = (int)pages.size() - from;
        pages.insert(pages.end(), s.pages.begin() + from, s.pages.begin() + to);
        return at;
    }

    void walk() {
        std::vector<Span> todo;
        todo.push_back({0, (int)nodes_.size(), 0, 0});
        while (!todo.empty()) {
            Span sp = todo.back();
            todo.pop_back();
            const Node &a = nodes_[sp.lo];
            if (sp.hi - sp.lo == 1) {
                const int len = a.seq->len, all = (len + pt_ - 1) / pt_;
                const int page_at = list_pages(*a.seq, sp.start, all);
                segs_.push_back({a.row0, a.n_new * shape_.group, sp.start * pt_, len, page_at, 1});
                continue;
            }
            // how far all of them agree: the sorted range's ends decide
            const Node &z = nodes_[sp.hi - 1];
            int most = z.shareable;
            for (int i = sp.lo; i < sp.hi; ++i) most = std::min(most, nodes_[i].shareable);
            const int d = agree(a, z, sp.depth, most);
            const int rows = z.row0 + z.n_new * shape_.group - a.row0;
            const long long run = (long long)(d - sp.start) * pt_;
            // Saved: the run's time for each sequence alone less that for all (chunks of many tokens, which are
            // bound by the products, save nothing); added: every row's partial result, written and read.
            long long apart = 0;
            for (int i = sp.lo; i < sp.hi; ++i) apart += cost(nodes_[i].n_new * shape_.group);
            if ((apart - cost(rows)) * run > (long long)rows * shape_.part_cost) {
                const int page_at = list_pages(*a.seq, sp.start, d);
                segs_.push_back({a.row0, rows, sp.start * pt_, d * pt_, page_at, 0});
                sp.start = d;
            }
            // children: neighbours that agree on the next page
            for (int lo = sp.lo; lo < sp.hi;) {
                int hi = lo + 1;
                if (nodes_[lo].shareable > d)
                    while (hi < sp.hi && nodes_[hi].shareable > d && nodes_[hi].seq->pages[d] == nodes_[lo].seq->pages[d])
                        ++hi;
                todo.push_back({lo, hi, sp.start, hi - lo > 1 ? d + 1 : d});
                lo = hi;
            }
        }
    }

    void cut(int rows) {
        long long total = 0;
        for (const Segment &s : segs_) total += cost(s.n_rows) * (s.key1 - s.key0);
        const long long target = std::max(1, shape_.workgroups / shape_.n_kv);
        const long long share = (total + target - 1) / target;  // of one workgroup
        // Pieces of about a workgroup's share each; somewhat longer ones where that ends earlier (24 ragged sequences
        // of up to 12000 f16 keys: 125 us with 74 pieces for 64 places, 114 with 64).
        std::vector<int> count(rows, 0);
        long long best = -1;
        int chosen = 0;
        for (int stretch : {100, 110, 120, 130, 150}) {
            const bool split = cut_all(share * stretch / 100, count);
            if (!split && best < 0) break;
            const long long end = makespan((int)target, count);
            if (best < 0 || end < best) {
                best = end;
                chosen = stretch;
            }
            if (!split) break;  // (longer pieces are the same)
        }
        if (best >= 0) cut_all(share * chosen / 100, count);
        // long pieces first: the short ones fill the end
        std::stable_sort(items.begin(), items.end(), [this](const AttnItem &a, const AttnItem &b) {
            return (long long)tile_cost(a.n_rows) * (a.key1 - a.key0) > (long long)tile_cost(b.n_rows) * (b.key1 - b.key0);
        });
        std::vector<int> start(rows + 1, 0);
        for (int r = 0; r < rows; ++r) {
            start[r + 1] = start[r] + (count[r] > 1 ? count[r] : 0);
            if (count[r] > 1) {
                join_rows.push_back(r);
                join_at.push_back(start[r]);
            }
        }
        join_at.push_back(start[rows]);
        join_parts.resize(start[rows]);
        // (a tile's rows all have the same pieces or more: any of them joined makes the item partial)
        std::vector<int> filled(rows, 0);
        for (AttnItem &it : items) {
            bool joined = false;
            for (int j = 0; j < it.n_rows; ++j) joined |= count[it.row0 + j] > 1;
            if (!joined) continue;
            it.part = parts;
            for (int j = 0; j < it.n_rows; ++j) {
                const int r = it.row0 + j;
                if (count[r] > 1) join_parts[start[r] + filled[r]++] = parts + j;
            }
            parts += it.n_rows;
        }
    }

    // The segments' pieces with this share of work each; whether any tile has more than one.
    bool cut_all(long long share, std::vector<int> &count) {
        items.clear();
        std::fill(count.begin(), count.end(), 0);
        size_t whole = 0;
        for (const Segment &s : segs_)
            for (int r = 0, nr; r < s.n_rows; r += nr, ++whole) {
                nr = tile(s.n_rows - r);
                cut_tile(s, r, nr, share, count);
            }
        return items.size() > whole;
    }

    // When the last workgroup ends if `places` of them take the items, the longest first, as they come free.
    long long makespan(int places, const std::vector<int> &count) {
        constexpr int kStart = 30000;  // a workgroup's first loads, 3 us
        costs_.clear();
        for (const AttnItem &it : items)
            costs_.push_back((long long)tile_cost(it.n_rows) * (it.key1 - it.key0) + kStart +
                             (count[it.row0] > 1 ? (long long)it.n_rows * shape_.part_cost : 0));
        std::sort(costs_.begin(), costs_.end(), std::greater<long long>());
        busy_.assign(std::min<size_t>(places, costs_.size()), 0);
        long long end = 0;
        for (long long c : costs_) {  // (a heap with the earliest end on top)
            std::pop_heap(busy_.begin(), busy_.end(), std::greater<long long>());
            busy_.back() += c;
            end = std::max(end, busy_.back());
            std::push_heap(busy_.begin(), busy_.end(), std::greater<long long>());
        }
        return end;
    }

    void cut_tile(const Segment &s, int r, int nr, long long share, std::vector<int> &count) {
        int key1 = s.key1;
        if (s.causal)  // the tile's last token sees no further than itself
            key1 = std::min(key1, tokens[(s.row0 + r + nr - 1) / shape_.group].order_pos + 1);
        const int keys = key1 - s.key0;
        const int least = std::min(256, std::max(64, shape_.min_cost / tile_cost(nr)));
        const long long piece = std::max<long long>(least, share / tile_cost(nr));
        // (one piece and no second kernel up to half more than the least)
        const int n = piece == least && keys <= least + least / 2 ? 1 : (int)((keys + piece - 1) / piece);
        const int step = ((keys + n - 1) / n + kKeyStep - 1) / kKeyStep * kKeyStep;
        for (int k = 0; k < keys; k += step) {
            items.push_back({s.row0 + r, nr, s.key0 + k, std::min(s.key0 + k + step, key1), s.page_at, s.causal, -1, 0});
            for (int j = 0; j < nr; ++j) count[s.row0 + r + j]++;
        }
    }

    const KvTables *kv_ = nullptr;
    PlanShape shape_{};
    int pt_ = 0;
    int best_[9] = {}, step_[9] = {};
    std::vector<Node> nodes_;
    std::vector<Segment> segs_;
    std::vector<long long> costs_, busy_;
};

}  // namespace exq
