// The routing of a step to experts, as its products see it.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"
#include "edgexpu_hip.h"

namespace exq {

constexpr int kMoeMaxExperts = 512, kMoeMaxTopK = 32, kMoeMaxGroups = 64;

// A tile of T places of the sorted pairs, all of one expert: the `index`-th of its
// expert's, from `start`, with `rest` pairs from there to the expert's end (none: no tile).
// Expert e's tiles begin at slot start_e / T + e: the next expert's are then past them
// whatever the counts, so no expert needs to know the others' tile counts.
struct MoeTile {
    int expert, start, rest, index;
};

}  // namespace exq

struct edgexpu_hip_moe {
    int n_experts = 0, top_k = 0, max_tokens = 0, n_embd = 0, n_ff = 0;
    int m = -1;     // tokens of the last routing that was queued (-1: none yet)
    int tile = 0;   // places a tile of its sorted pairs (32 or 64); 0: not sorted
    uint8_t *mem = nullptr;
    // Tokens of the last routing that ran, which replays of captured ones make another than the last queued
    // (-1: none yet, or one whose pairs are still to be sorted).  What a routing leaves in ids, order and tiles
    // follows from its tokens, so that a product reads them only where the two are equal.
    int32_t *routed = nullptr;
    int32_t *ids = nullptr;  // [max_tokens][top_k], -1: no expert
    float *weights = nullptr;
    int32_t *order = nullptr;       // pairs (token * top_k + place) by expert, then by number
    exq::MoeTile *tiles = nullptr;
    uint8_t *pack = nullptr;        // quantized activations of the product at hand
    float *part = nullptr;          // [max_tokens][top_k][n_embd]: a token's parts of the down product
    size_t pairs() const { return (size_t)(m > 0 ? m : 0) * top_k; }
};

namespace exq {

struct RouteArgs {
    const float *scores, *bias;
    int32_t *ids, *ids_out, *routed;
    float *weights, *weights_out;
    int now;  // what `routed` becomes
    int m, n_experts, top_k, sigmoid, n_groups, top_groups, group_best, normalise;
    double scale;
};

hipError_t launch_moe_route(const RouteArgs &a, hipStream_t st);
// (no pairs: `routed` alone is written)
hipError_t launch_moe_assign(const int32_t *ids, const float *weights, int32_t *to_ids, float *to_weights, int pairs,
                             int n_experts, int32_t *routed, int now, hipStream_t st);
// Sorts the pairs by expert into tiles of T places: moe_slots(pairs, n_experts, T) slots are written.  *routed = m.
hipError_t launch_moe_sort(const int32_t *ids, int pairs, int n_experts, int T, int32_t *order, MoeTile *tiles,
                           int32_t *routed, int m, hipStream_t st);
inline int moe_slots(long long pairs, int n_experts, int T) { return (int)(pairs / T) + n_experts; }

}  // namespace exq
