// Routing to experts: each token's top_k of n_experts by its scores.
//
//   p = softmax(s) or 1 / (1 + exp(-s));  c = p + bias
//   groups of experts ranked by their best one or two c, the best groups stay
//   the top_k largest c, ties to the lowest index; weight = p [/ sum p] * scale
//
// All of it in 64 bits: which expert is chosen depends on which of two nearly
// equal values is larger, and f32 sums round differently in every order.  The
// work is small (a score is 4 bytes and one exponential), so that costs little.
//
// One wave a token: lane l holds experts l, l + 64, ..., so a row is read in
// whole lines.
#include <cmath>

#include "moe.h"

namespace exq {

constexpr int kRouteWaves = 4;
constexpr int kRouteSlots = kMoeMaxExperts / 64;

// A double's order as an unsigned integer's (minus infinity above zero; 0 is below every number).
__device__ __forceinline__ uint64_t order_key(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}
constexpr uint64_t kNoKey = 0;  // not to be chosen

__device__ __forceinline__ uint64_t shfl_xor_u64(uint64_t v, int off) {
    const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)v, off, 64);
    const uint32_t hi = (uint32_t)__shfl_xor((int)(uint32_t)(v >> 32), off, 64);
    return (uint64_t)lo | ((uint64_t)hi << 32);
}
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const uint64_t o = shfl_xor_u64(v, off);
        v = o > v ? o : v;
    }
    return v;
}
__device__ __forceinline__ int wave_min_i32(int v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = min(v, __shfl_xor(v, off, 64));
    return v;
}
__device__ __forceinline__ double read_lane_f64(double v, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)b, lane, 64);
    const uint32_t hi = (uint32_t)__shfl((int)(uint32_t)(b >> 32), lane, 64);
    return __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
}

__global__ __launch_bounds__(64 * kRouteWaves) void moe_route_kernel(RouteArgs a) {
    __shared__ double cs[kRouteWaves][kMoeMaxExperts];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // (a wave past the last token repeats it and writes nothing: all reach the barrier)
    const bool mine_t = (int)blockIdx.x * kRouteWaves + wave < a.m;
    const int t = mine_t ? (int)blockIdx.x * kRouteWaves + wave : a.m - 1;
    const float *s = a.scores + (size_t)t * a.n_experts;
    double p[kRouteSlots];
    bool live[kRouteSlots];
    double top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kRouteSlots; ++i) {
        const int e = lane + 64 * i;
        p[i] = e < a.n_experts ? (double)s[e] : INFINITY;
        live[i] = fabs(p[i]) < INFINITY;
        if (live[i]) top = fmax(top, p[i]);
    }
    if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < kRouteSlots; ++i) p[i] = live[i] ? 1.0 / (1.0 + exp(-p[i])) : 0.0;
    } else {
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            const uint64_t o = shfl_xor_u64(__builtin_bit_cast(uint64_t, top), off);
            top = fmax(top, __builtin_bit_cast(double, o));
        }
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < kRouteSlots; ++i) {
            p[i] = live[i] ? exp(p[i] - top) : 0.0;
            sum += p[i];
        }
        sum = wave_sum_f64(sum);  // (0 only where no score is live)
#pragma unroll
        for (int i = 0; i < kRouteSlots; ++i) p[i] = live[i] ? p[i] / sum : 0.0;
    }
    uint64_t key[kRouteSlots];
#pragma unroll
    for (int i = 0; i < kRouteSlots; ++i) {
        const int e = lane + 64 * i;
        const double c = live[i] && a.bias != nullptr ? p[i] + (double)a.bias[e] : p[i];
        key[i] = live[i] && fabs(c) < INFINITY ? order_key(c) : kNoKey;
        if (a.n_groups > 1 && e < a.n_experts) cs[wave][e] = key[i] != kNoKey ? c : -INFINITY;
    }
    if (a.n_groups > 1) {
        // lane g ranks group g
        __syncthreads();
        const int per = a.n_experts / a.n_groups;
        double b0 = -INFINITY, b1 = -INFINITY;
        if (lane < a.n_groups)
            for (int i = 0; i < per; ++i) {
                const double c = cs[wave][lane * per + i];
                if (c > b0) {
                    b1 = b0;
                    b0 = c;
                } else if (c > b1) {
                    b1 = c;
                }
            }
        const double rank = a.group_best == 2 && b1 > -INFINITY ? b0 + b1 : b0;
        int ahead = 0;
        for (int g = 0; g < a.n_groups; ++g) {
            const double o = read_lane_f64(rank, g);
            ahead += o > rank || (o == rank && g < lane) ? 1 : 0;
        }
        const unsigned long long stay = __ballot(lane < a.n_groups && ahead < a.top_groups);
#pragma unroll
        for (int i = 0; i < kRouteSlots; ++i) {
            const int e = lane + 64 * i;
            if (e < a.n_experts && !((stay >> (e / per)) & 1ull)) key[i] = kNoKey;
        }
    }
    // the choices, one after the other; lane j keeps the j-th
    int id = -1;
    double w = 0.0, total = 0.0;
    for (int j = 0; j < a.top_k; ++j) {
        uint64_t best = kNoKey;
#pragma unroll
        for (int i = 0; i < kRouteSlots; ++i) best = key[i] > best ? key[i] : best;
        const uint64_t all = wave_max_u64(best);
        if (all == kNoKey) break;  // (the same in every lane)
        int mine = kMoeMaxExperts;
#pragma unroll
        for (int i = kRouteSlots - 1; i >= 0; --i)
            if (key[i] == all) mine = lane + 64 * i;
        const int e = wave_min_i32(mine);
        double pe = 0.0;
#pragma unroll
        for (int i = 0; i < kRouteSlots; ++i)
            if (lane + 64 * i == e) {
                key[i] = kNoKey;
                pe = p[i];
            }
        pe = read_lane_f64(pe, e & 63);
        total += pe;
        if (lane == j) {
            id = e;
            w = pe;
        }
    }
    if (mine_t && lane < a.top_k) {
        if (a.normalise && total > 0.0) w /= total;
        const float wf = (float)(w * a.scale);
        const size_t at = (size_t)t * a.top_k + lane;
        a.ids[at] = id;
        a.weights[at] = id >= 0 ? wf : 0.0f;
        if (a.ids_out != nullptr) a.ids_out[at] = id;
        if (a.weights_out != nullptr) a.weights_out[at] = id >= 0 ? wf : 0.0f;
    }
}

__global__ __launch_bounds__(256) void moe_assign_kernel(const int32_t *__restrict__ ids,
                                                         const float *__restrict__ weights, int32_t *to_ids,
                                                         float *to_weights, int pairs, int n_experts) {
    const int i = (int)(blockIdx.x * 256 + threadIdx.x);
    if (i >= pairs) return;
    const int e = ids[i];
    const bool some = e >= 0 && e < n_experts;
    to_ids[i] = some ? e : -1;
    to_weights[i] = some ? weights[i] : 0.0f;
}

// Pairs by expert: a workgroup an expert counts the pairs of the experts before its
// own, then writes its own pairs in ascending order (so the sort is stable and the
// same every time) and its tiles.  Every workgroup reads all ids, 4 bytes a pair from
// L2, and none waits for another.
constexpr int kSortThreads = 1024, kSortEach = 8;  // (ids are read 8 a thread)
struct Ids8 {
    int v[kSortEach];
};
// Pairs first .. + 7, those past the last as no pair's id.
__device__ __forceinline__ Ids8 load_ids(const int32_t *ids, int first, int pairs) {
    Ids8 r;
    const int4 *p = reinterpret_cast<const int4 *>(ids + first);
    const int4 none = make_int4(-1, -1, -1, -1);
    const int4 a = first < pairs ? p[0] : none, b = first + 4 < pairs ? p[1] : none;
    const int v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int k = 0; k < 8; ++k) r.v[k] = first + k < pairs ? v[k] : -1;
    return r;
}
__global__ __launch_bounds__(kSortThreads) void moe_sort_kernel(const int32_t *__restrict__ ids, int pairs,
                                                                int n_experts, int T, int slots,
                                                                int32_t *__restrict__ order,
                                                                MoeTile *__restrict__ tiles) {
    constexpr int kWaves = kSortThreads / 64, kRound = kSortThreads * kSortEach, kKeep = 4;
    __shared__ int sums[2][kWaves];
    const int e = (int)blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    Ids8 kept[kKeep];  // the first rounds' ids stay in registers for the second pass
    int less = 0, own = 0;
#pragma unroll
    for (int i = 0; i < kKeep; ++i) kept[i] = load_ids(ids, i * kRound + tid * kSortEach, pairs);
    const auto count = [&](const Ids8 &c) {
#pragma unroll
        for (int k = 0; k < kSortEach; ++k) {
            less += c.v[k] >= 0 && c.v[k] < e ? 1 : 0;
            own += c.v[k] == e ? 1 : 0;
        }
    };
#pragma unroll
    for (int i = 0; i < kKeep; ++i) count(kept[i]);
    for (int i0 = kKeep * kRound; i0 < pairs; i0 += kRound) count(load_ids(ids, i0 + tid * kSortEach, pairs));
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        less += __shfl_xor(less, off, 64);
        own += __shfl_xor(own, off, 64);
    }
    if (lane == 0) {
        sums[0][wave] = less;
        sums[1][wave] = own;
    }
    __syncthreads();
    less = own = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        less += sums[0][w];
        own += sums[1][w];
    }
    const int slot0 = less / T + e, slot1 = e + 1 < n_experts ? (less + own) / T + e + 1 : slots;
    for (int s = slot0 + tid; s < slot1; s += kSortThreads) {
        const int at = (s - slot0) * T;
        tiles[s] = MoeTile{e, less + at, max(0, own - at), s - slot0};
    }
    int base = less;
    // (every thread runs the same rounds: base and own are the workgroup's)
    const auto place = [&](const Ids8 &c, int first) {
        unsigned hit = 0u;
#pragma unroll
        for (int k = 0; k < kSortEach; ++k)
            if (c.v[k] == e) hit |= 1u << k;
        const int mine = __popc(hit);
        int before = mine;  // inclusive over the wave, then over the waves
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int o = __shfl_up(before, off, 64);
            if (lane >= off) before += o;
        }
        __syncthreads();  // (the sums of the round before have been read)
        if (lane == 63) sums[0][wave] = before;
        __syncthreads();
        int at = base + before - mine, total = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            at += w < wave ? sums[0][w] : 0;
            total += sums[0][w];
        }
#pragma unroll
        for (int k = 0; k < kSortEach; ++k)
            if ((hit >> k) & 1u) order[at++] = first + k;
        base += total;
    };
#pragma unroll
    for (int i = 0; i < kKeep; ++i)
        if (i * kRound < pairs && base < less + own) place(kept[i], i * kRound + tid * kSortEach);
    for (int i0 = kKeep * kRound; i0 < pairs && base < less + own; i0 += kRound)
        place(load_ids(ids, i0 + tid * kSortEach, pairs), i0 + tid * kSortEach);
}

hipError_t launch_moe_sort(const int32_t *ids, int pairs, int n_experts, int T, int32_t *order, MoeTile *tiles,
                           hipStream_t st) {
    hipLaunchKernelGGL(moe_sort_kernel, dim3((unsigned)n_experts), dim3(kSortThreads), 0, st, ids, pairs, n_experts, T,
                       moe_slots(pairs, n_experts, T), order, tiles);
    return hipGetLastError();
}

hipError_t launch_moe_route(const RouteArgs &a, hipStream_t st) {
    const dim3 grid((unsigned)((a.m + kRouteWaves - 1) / kRouteWaves));
    hipLaunchKernelGGL(moe_route_kernel, grid, dim3(64 * kRouteWaves), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_moe_assign(const int32_t *ids, const float *weights, int32_t *to_ids, float *to_weights, int pairs,
                             int n_experts, hipStream_t st) {
    hipLaunchKernelGGL(moe_assign_kernel, dim3((unsigned)((pairs + 255) / 256)), dim3(256), 0, st, ids, weights, to_ids,
                       to_weights, pairs, n_experts);
    return hipGetLastError();
}

}  // namespace exq
