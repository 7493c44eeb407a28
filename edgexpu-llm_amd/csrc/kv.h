// The paged cache's and the step's handles, and how kernels see them.
#pragma once

#include <hip/hip_runtime.h>

#include <vector>

#include "attn_plan.h"
#include "common.h"
#include "edgexpu_hip.h"
#include "kv_tables.h"

struct edgexpu_hip_kv {
    edgexpu_hip_kv(int page_tokens, int n_pages, int max_seqs) : tables(page_tokens, n_pages, max_seqs) {}
    exq::KvTables tables;
    int type = 0, n_layers = 0, n_kv = 0, dim = 0;
    size_t head_bytes = 0;  // one head's K or V of a page
    uint8_t *pool = nullptr;
    bool owned = false;
    int n_batches = 0;
    std::vector<exq::KvMove> moves;
    size_t page_bytes() const { return 2 * (size_t)n_kv * head_bytes; }
    size_t layer_bytes() const { return (size_t)tables.n_pages() * page_bytes(); }
};

struct edgexpu_hip_batch {
    edgexpu_hip_kv *kv = nullptr;
    int n_heads = 0, max_seqs = 0, max_tokens = 0;
    exq::AttnPlan plan, made;  // made: of the set at hand, the plan once nothing refuses it
    bool set = false;
    uint64_t epoch = 0;     // the tables' when the plan was made
    bool captured = false;  // a captured call holds the device pointers
    int captured_tokens = INT32_MAX;  // the fewest that the buffers of a captured call hold
    bool captured_append = false;     // a captured call writes to the plan's slots
    // device plan, 32-bit words: the tokens backwards (token t in the four
    // words before head - 4 * t), so that they and what follows are one copy;
    // from `head` on the header, the items, the pages, the joins
    int32_t *words = nullptr;
    size_t words_cap = 0;  // behind head
    int32_t *head() const { return words + 4 * (size_t)max_tokens; }
    float *part = nullptr;  // partial results: [part][kv head][dim], then (maximum, sum) pairs
    size_t part_cap = 0;    // partial results of all kv heads
    // host copies in flight
    static constexpr int kStages = 4;
    int32_t *stage[kStages] = {};
    size_t stage_cap[kStages] = {};
    hipEvent_t done[kStages] = {};
    bool busy[kStages] = {};
    int next = 0;
};

namespace exq {

// One layer of the pool.  slot = page * page_tokens + offset; a head's row of
// K (which = 0) or V (1) lies at
//   base + page * page_bytes + (which * n_kv + head) * head_bytes + offset * row bytes.
struct KvView {
    uint8_t *base;
    size_t page_bytes;
    unsigned head_bytes;
    int page_shift, n_kv;
};

inline int log2i(int v) { return 31 - __builtin_clz((unsigned)v); }

inline KvView kv_view(const edgexpu_hip_kv *kv, int layer) {
    return {kv->pool + (size_t)layer * kv->layer_bytes(), kv->page_bytes(), (unsigned)kv->head_bytes,
            log2i(kv->tables.page_tokens()), kv->n_kv};
}

// false (sticky error) unless the batch is set, fresh and `layer` exists; *capturing: the call is being recorded.
bool batch_ready(edgexpu_hip_batch *b, int layer, hipStream_t st, const char *what, bool *capturing);
// A call that nothing refuses any more is about to be recorded: the batch keeps the buffers that it holds.
void batch_recorded(edgexpu_hip_batch *b);

// attn.hip: how many of its kernel's workgroups run at once.
int attn_workgroups(int type, int dim);
// Allows the kernel the LDS it takes (once for a batch: nothing of it is left for a captured call).
hipError_t attn_prepare(int type, int dim);

}  // namespace exq
