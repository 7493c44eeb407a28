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
#include <algorithm>
#include <cmath>

#include "moe.h"

namespace exq {

constexpr int kRouteWaves = 4;

// A double's order as an unsigned integer's.  0 is below every number's key, and so is
// every key whose high word is 0.
__device__ __forceinline__ uint64_t order_key(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}

// Reductions over the wave by DPP (row shifts, then row broadcasts: the total arrives in
// lane 63): a step is a few cycles, where one through LDS is a hundred, and a token's
// choices are one chain of them.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_from(uint32_t old, uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)old, (int)v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    v = max(v, dpp_from<0x111, 0xf>(v, v));
    v = max(v, dpp_from<0x112, 0xf>(v, v));
    v = max(v, dpp_from<0x114, 0xf>(v, v));
    v = max(v, dpp_from<0x118, 0xf>(v, v));
    v = max(v, dpp_from<0x142, 0xa>(v, v));
    v = max(v, dpp_from<0x143, 0xc>(v, v));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ double lane_f64(double v, int lane) {  // (lane: the same in the whole wave)
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double v) {  // (lanes without a source add 0)
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = dpp_from<CTRL, ROWS>(0u, (uint32_t)b), hi = dpp_from<CTRL, ROWS>(0u, (uint32_t)(b >> 32));
    return v + __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
}
__device__ __forceinline__ double wave_add_f64(double v) {
    v = dpp_add<0x111, 0xf>(v);
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);
    v = dpp_add<0x143, 0xc>(v);
    return lane_f64(v, 63);
}
__device__ __forceinline__ double shfl_xor_f64(double v, int off) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)b, off, 64);
    const uint32_t hi = (uint32_t)__shfl_xor((int)(uint32_t)(b >> 32), off, 64);
    return __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
}

// S = ceil(n_experts / 64) experts a lane.  Bound by the chain of a wave: 64-bit exponentials and one
// choice after the other (1 token, 8 of 128, 4.1 us; 4096 tokens, 8 of 256 in groups, 12 us).
template <int S>
__global__ __launch_bounds__(64 * kRouteWaves) void moe_route_kernel(RouteArgs a) {
    __shared__ double cs[kRouteWaves][64 * S];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // (a wave past the last token repeats it and writes nothing: all reach the barrier)
    const bool own = (int)blockIdx.x * kRouteWaves + wave < a.m;
    const int t = own ? (int)blockIdx.x * kRouteWaves + wave : a.m - 1;
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.routed = a.now;
    const float *s = a.scores + (size_t)t * a.n_experts;
    float sc[S];
    bool live[S];
    uint32_t top = 0u;  // the largest live score's order
#pragma unroll
    for (int i = 0; i < S; ++i) {
        const int e = lane + 64 * i;
        sc[i] = e < a.n_experts ? s[e] : INFINITY;
        live[i] = fabsf(sc[i]) < INFINITY;
        const uint32_t b = __float_as_uint(sc[i]);
        if (live[i]) top = max(top, (b >> 31) ? ~b : b | 0x80000000u);
    }
    double p[S];
    if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < S; ++i) p[i] = live[i] ? 1.0 / (1.0 + exp(-(double)sc[i])) : 0.0;
    } else {
        top = wave_max_u32(top);
        const double mx = (double)__uint_as_float((top >> 31) ? top & 0x7fffffffu : ~top);
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            p[i] = live[i] ? exp((double)sc[i] - mx) : 0.0;
            sum += p[i];
        }
        const double inv = 1.0 / wave_add_f64(sum);  // (the sum is 0 only where no score is live)
#pragma unroll
        for (int i = 0; i < S; ++i) p[i] = live[i] ? p[i] * inv : 0.0;
    }
    uint32_t hi[S], lo[S];  // the choice's keys
#pragma unroll
    for (int i = 0; i < S; ++i) {
        const int e = lane + 64 * i;
        const double c = live[i] && a.bias != nullptr ? p[i] + (double)a.bias[e] : p[i];
        const bool open = live[i] && fabs(c) < INFINITY;
        const uint64_t key = open ? order_key(c) : 0ull;
        hi[i] = (uint32_t)(key >> 32);
        lo[i] = (uint32_t)key;
        if (a.n_groups > 1) cs[wave][e] = open ? c : -INFINITY;
    }
    if (a.n_groups > 1) {
        __syncthreads();
        // `width` lanes a group, each over its share of the group's values
        const int per = a.n_experts / a.n_groups, log = 31 - __clz(64 / a.n_groups), width = 1 << log;
        const int mine = lane >> log;
        double b0 = -INFINITY, b1 = -INFINITY;
        const auto take = [&](double c) {
            b1 = fmax(b1, fmin(b0, c));
            b0 = fmax(b0, c);
        };
        if (mine < a.n_groups)
            for (int i = lane & (width - 1); i < per; i += width) take(cs[wave][mine * per + i]);
        for (int off = width >> 1; off > 0; off >>= 1) {
            const double o0 = shfl_xor_f64(b0, off), o1 = shfl_xor_f64(b1, off);
            take(o0);
            take(o1);
        }
        const double rank = a.group_best == 2 && b1 > -INFINITY ? b0 + b1 : b0;
        int ahead = 0;
        for (int g = 0; g < a.n_groups; ++g) {
            const double o = lane_f64(rank, g << log);
            ahead += o > rank || (o == rank && g < mine) ? 1 : 0;
        }
        const unsigned long long stay = __ballot(mine < a.n_groups && ahead < a.top_groups);
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const int e = lane + 64 * i;
            if (e < a.n_experts && !((stay >> ((e / per) << log)) & 1ull)) hi[i] = lo[i] = 0u;
        }
    }
    // The choices, one after the other; lane j keeps the j-th.  The largest high word
    // mostly says which; where several have it, the largest low word among them, and
    // of equals the first slot's first lane, the lowest number.
    int id = -1;
    double w = 0.0, total = 0.0;
    for (int j = 0; j < a.top_k; ++j) {
        uint32_t best = hi[0];
#pragma unroll
        for (int i = 1; i < S; ++i) best = max(best, hi[i]);
        const uint32_t H = wave_max_u32(best);
        if (H == 0u) break;
        unsigned long long has[S];
        int n = 0;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            has[i] = __ballot(hi[i] == H);
            n += __popcll(has[i]);
        }
        if (n > 1) {
            uint32_t low = 0u;
#pragma unroll
            for (int i = 0; i < S; ++i)
                if (hi[i] == H) low = max(low, lo[i]);
            const uint32_t L = wave_max_u32(low);
#pragma unroll
            for (int i = 0; i < S; ++i) has[i] &= __ballot(lo[i] == L);
        }
        int slot = S - 1;
        double ps = p[S - 1];
        unsigned long long first = has[S - 1];
#pragma unroll
        for (int i = S - 2; i >= 0; --i)
            if (has[i] != 0ull) {
                slot = i;
                ps = p[i];
                first = has[i];
            }
        const int at = __ffsll((long long)first) - 1;
        const double pe = lane_f64(ps, at);
        total += pe;
        if (lane == j) {
            id = 64 * slot + at;
            w = pe;
        }
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (slot == i && lane == at) hi[i] = lo[i] = 0u;
    }
    if (own && lane < a.top_k) {
        if (a.normalise && total > 0.0) w /= total;
        const float wf = id >= 0 ? (float)(w * a.scale) : 0.0f;
        const size_t at = (size_t)t * a.top_k + lane;
        a.ids[at] = id;
        a.weights[at] = wf;
        if (a.ids_out != nullptr) a.ids_out[at] = id;
        if (a.weights_out != nullptr) a.weights_out[at] = wf;
    }
}

__global__ __launch_bounds__(256) void moe_assign_kernel(const int32_t *__restrict__ ids,
                                                         const float *__restrict__ weights, int32_t *to_ids,
                                                         float *to_weights, int pairs, int n_experts,
                                                         int32_t *routed, int now) {
    const int i = (int)(blockIdx.x * 256 + threadIdx.x);
    if (i == 0) *routed = now;
    if (i >= pairs) return;
    const int e = ids[i];
    const bool some = e >= 0 && e < n_experts;
    to_ids[i] = some ? e : -1;
    to_weights[i] = some ? weights[i] : 0.0f;
}

// Pairs by expert: a workgroup an expert counts the pairs of the experts before its
// own, then writes its own pairs in ascending order (so the sort is stable and the
// same every time) and its tiles.  Every workgroup reads all ids, 4 bytes a pair from
// L2, and none waits for another (32768 pairs of 256 experts 9 us; a token's 5).
constexpr int kSortThreads = 1024, kSortMost = 32;  // ids a thread and round, read 4 at once
__global__ __launch_bounds__(kSortThreads) void moe_sort_kernel(const int32_t *__restrict__ ids, int pairs,
                                                                int n_experts, int T, int slots, int each,
                                                                int32_t *__restrict__ order,
                                                                MoeTile *__restrict__ tiles, int32_t *routed, int m) {
    constexpr int kWaves = kSortThreads / 64;
    __shared__ int sums[2][kWaves];
    const int e = (int)blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int round = each * kSortThreads;
    if (e == 0 && tid == 0) *routed = m;
    // A thread's ids of a round from `first` on (each of them, those past the last as -1):
    // which are this expert's, and how many are of those before it.
    const auto read = [&](int first, int &less) {
        int4 v[kSortMost / 4];
#pragma unroll
        for (int j = 0; j < kSortMost / 4; ++j)
            v[j] = 4 * j < each && first + 4 * j < pairs ? *reinterpret_cast<const int4 *>(ids + first + 4 * j)
                                                         : make_int4(-1, -1, -1, -1);
        unsigned hit = 0u;
#pragma unroll
        for (int j = 0; j < kSortMost / 4; ++j) {
            const int q[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int id = first + 4 * j + k < pairs ? q[k] : -1;
                less += (unsigned)id < (unsigned)e ? 1 : 0;
                hit |= id == e ? 1u << (4 * j + k) : 0u;
            }
        }
        return hit;
    };
    int less = 0, own = 0;
    const unsigned hit0 = read(tid * each, less);
    own = __popc(hit0);
    for (int i0 = round; i0 < pairs; i0 += round) own += __popc(read(i0 + tid * each, less));
    int before = __popc(hit0);  // of the first round: inclusive over the wave
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(before, off, 64);
        if (lane >= off) before += o;
    }
    __shared__ int first_sums[kWaves];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        less += __shfl_xor(less, off, 64);
        own += __shfl_xor(own, off, 64);
    }
    if (lane == 63) {
        sums[0][wave] = less;
        sums[1][wave] = own;
        first_sums[wave] = before;
    }
    __syncthreads();
    less = own = 0;
    int at = before - __popc(hit0), total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        less += sums[0][w];
        own += sums[1][w];
        at += w < wave ? first_sums[w] : 0;
        total += first_sums[w];
    }
    const int slot0 = less / T + e, slot1 = e + 1 < n_experts ? (less + own) / T + e + 1 : slots;
    for (int s = slot0 + tid; s < slot1; s += kSortThreads) {
        const int from = (s - slot0) * T;
        tiles[s] = MoeTile{e, less + from, max(0, own - from), s - slot0};
    }
    const auto place = [&](unsigned hit, int first, int to) {
        while (hit != 0u) {
            order[to++] = first + __ffs((int)hit) - 1;
            hit &= hit - 1u;
        }
    };
    place(hit0, tid * each, less + at);
    int base = less + total;
    for (int i0 = round; i0 < pairs && base < less + own; i0 += round) {  // (the same rounds in every thread)
        int unused = 0;
        const unsigned hit = read(i0 + tid * each, unused);
        int upto = __popc(hit);
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int o = __shfl_up(upto, off, 64);
            if (lane >= off) upto += o;
        }
        __syncthreads();  // (the sums of the round before have been read)
        if (lane == 63) first_sums[wave] = upto;
        __syncthreads();
        int to = base + upto - __popc(hit);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            to += w < wave ? first_sums[w] : 0;
            base += first_sums[w];
        }
        place(hit, i0 + tid * each, to);
    }
}

hipError_t launch_moe_sort(const int32_t *ids, int pairs, int n_experts, int T, int32_t *order, MoeTile *tiles,
                           int32_t *routed, int m, hipStream_t st) {
    const int each = std::min(kSortMost, (pairs + 4 * kSortThreads - 1) / (4 * kSortThreads) * 4);
    hipLaunchKernelGGL(moe_sort_kernel, dim3((unsigned)n_experts), dim3(kSortThreads), 0, st, ids, pairs, n_experts, T,
                       moe_slots(pairs, n_experts, T), each, order, tiles, routed, m);
    return hipGetLastError();
}

hipError_t launch_moe_route(const RouteArgs &a, hipStream_t st) {
    const dim3 grid((unsigned)((a.m + kRouteWaves - 1) / kRouteWaves));
    const auto k = a.n_experts <= 64    ? moe_route_kernel<1>
                   : a.n_experts <= 128 ? moe_route_kernel<2>
                   : a.n_experts <= 256 ? moe_route_kernel<4>
                                        : moe_route_kernel<8>;
    hipLaunchKernelGGL(k, grid, dim3(64 * kRouteWaves), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_moe_assign(const int32_t *ids, const float *weights, int32_t *to_ids, float *to_weights, int pairs,
                             int n_experts, int32_t *routed, int now, hipStream_t st) {
    hipLaunchKernelGGL(moe_assign_kernel, dim3((unsigned)std::max(1, (pairs + 255) / 256)), dim3(256), 0, st, ids,
                       weights, to_ids, to_weights, pairs, n_experts, routed, now);
    return hipGetLastError();
}

}  // namespace exq
