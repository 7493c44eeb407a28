// The attention plan with the costs of csrc/attn_plan.h, behind C functions for test_attn_costs.py.
#include "attn_plan.h"

using namespace exq;

extern "C" {
void costs(int type, int dim, int *of) {
    const RowCost c = attn_cost(type, dim);
    for (int k = 0; k < 4; ++k) of[k] = c.of[k];
}
// The rows of each of the items that `tokens` tokens of one sequence of `length` make; returns how many.
int item_rows(int type, int dim, int group, int length, int tokens, int *rows, int room) {
    KvTables kv(64, length / 64 + 1, 1);
    std::vector<KvMove> moves;
    const int s = kv.new_seq();
    if (kv.extend(1, &s, &length, moves) != KvStatus::ok) return -1;
    AttnPlan plan;
    plan.build(kv, 1, &s, &tokens, {group, 1, attn_cost(type, dim), (dim + 2) * 8, 512, 80000});
    for (size_t i = 0; i < plan.items.size() && (int)i < room; ++i) rows[i] = plan.items[i].n_rows;
    return (int)plan.items.size();
}
}
