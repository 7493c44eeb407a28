// The paged cache's bookkeeping and the attention plan (csrc/kv_tables.h,
// csrc/attn_plan.h), plain C++, behind C functions for test_kv_host.py.
#include <cstring>

#include "attn_plan.h"

using namespace exq;

namespace {
struct Host {
    Host(int page, int pages, int seqs) : kv(page, pages, seqs) {}
    KvTables kv;
    std::vector<KvMove> moves;
    AttnPlan plan;
};
}  // namespace

extern "C" {
Host *host_new(int page, int pages, int seqs) { return new Host(page, pages, seqs); }
void host_free(Host *h) { delete h; }
int host_seq(Host *h) { return h->kv.new_seq(); }
int host_fork(Host *h, int n, const int *p, int copy, int *c) {
    h->moves.clear();
    return (int)h->kv.fork(n, p, copy != 0, c, h->moves);
}
int host_extend(Host *h, int n, const int *s, const int *k) {
    h->moves.clear();
    return (int)h->kv.extend(n, s, k, h->moves);
}
int host_truncate(Host *h, int s, int n) { return (int)h->kv.truncate(s, n); }
int host_release(Host *h, int n, const int *s) { return (int)h->kv.release(n, s); }
int host_compact(Host *h) {
    h->moves.clear();
    return h->kv.compact(h->moves);
}
int host_free_pages(Host *h) { return h->kv.free_pages(); }
int host_moves(Host *h, int *out) {
    if (out) memcpy(out, h->moves.data(), h->moves.size() * sizeof(KvMove));
    return (int)h->moves.size();
}
int host_len(Host *h, int s) { return h->kv.valid(s) ? h->kv.seq(s).len : -1; }
int host_pages(Host *h, int s, int *out) {
    const std::vector<int> &p = h->kv.seq(s).pages;
    if (out && !p.empty()) memcpy(out, p.data(), p.size() * sizeof(int));
    return (int)p.size();
}
void host_plan(Host *h, int n, const int *s, const int *k, int group, int n_kv, const int *cost, int part_cost, int wgs) {
    h->plan.build(h->kv, n, s, k, {group, n_kv, {{cost[0], cost[1], cost[2], cost[3]}}, part_cost, wgs, 12000});
}
// 0 tokens (4 words each), 1 items (8), 2 pages, 3 join_rows, 4 join_at, 5 join_parts, 6 parts and writable
int host_plan_get(Host *h, int what, int *out) {
    const AttnPlan &p = h->plan;
    const auto give = [out](const void *d, size_t words) {
        if (out && words) memcpy(out, d, words * 4);
        return (int)words;
    };
    switch (what) {
        case 0: return give(p.tokens.data(), p.tokens.size() * 4);
        case 1: return give(p.items.data(), p.items.size() * 8);
        case 2: return give(p.pages.data(), p.pages.size());
        case 3: return give(p.join_rows.data(), p.join_rows.size());
        case 4: return give(p.join_at.data(), p.join_at.size());
        case 5: return give(p.join_parts.data(), p.join_parts.size());
        default: {
            const int v[2] = {p.parts, p.writable ? 1 : 0};
            return give(v, 2);
        }
    }
}
}
