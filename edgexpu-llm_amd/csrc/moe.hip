// The products of a step's tokens with the experts they were routed to.
//
//   act[t][j] = f(b_g[e] + W_g[e] . q8(x[t])) * (b_u[e] + W_u[e] . q8(x[t]))
//   out[t]    = [residual[t] +] sum_j w[t][j] (b[e] + W[e] . q8(act[t][j]))
//   e = ids[t][j]
#include <algorithm>
#include <cmath>
#include <new>

#include "lib.h"
#include "moe.h"
#include "moe_formats.h"

namespace exq {

__device__ __forceinline__ float gelu_f32(float v) {
    // v (1 + tanh u) / 2 = v / (1 + exp(-2 u)), which has no difference of near numbers
    const float u = v * fmaf(0.044715f * v, v, 1.0f) * 1.5957691216057308f;
    return v / (1.0f + expf(-u));
}
__device__ __forceinline__ float moe_act(float v, int activation) {
    return activation == EDGEXPU_HIP_MOE_GELU ? gelu_f32(v) : silu_f32(v);
}

struct MoeArgs {
    const int32_t *ids;
    const float *weights;
    const int32_t *order;
    const MoeTile *tiles;
    const uint8_t *w[2];      // gate and up, or down
    const float *bias[2];
    const float *x;           // f32 rows
    uint8_t *pack;            // their records, `groups` a row
    size_t row_bytes, expert_bytes;
    float *out;               // gate_up: act; down: out, or the pairs' parts
    const float *residual;
    int m, top_k, rows;       // weight rows of an expert
    int n, groups, nblk;      // elements of a row, its groups of 256, its blocks
    int activation;
};

// ------------------------------------------------------------------ packing

// Rows of x into records, 256 threads over a part of a row (blockIdx.y).  ACT: rows are
// tokens, and the places of a token that have no expert get zeros in `out` by the way.
template <bool K, bool ACT>
__global__ __launch_bounds__(256) void moe_pack_kernel(MoeArgs a) {
    const size_t row = blockIdx.x;
    const int part = (int)blockIdx.y * 256 + (int)threadIdx.x;
    if (part < moe_pack_parts<K>(a.n))
        moe_pack_part<K>(a.x + row * a.n, a.n, part, a.pack + row * a.groups * kMoeRec);
    if (ACT && blockIdx.y == 0)
        for (int j = 0; j < a.top_k; ++j) {
            const size_t pair = row * a.top_k + j;
            if (a.ids[pair] < 0)
                for (int i = threadIdx.x; i < a.rows; i += 256) a.out[pair * a.rows + i] = 0.0f;
        }
}

// ------------------------------------------------------------------ one token
//
// A workgroup takes 16 rows (gate and up: of each) for one token: of one of its
// experts (gate and up), or of all of them, whose weighted sum then needs no second
// launch (down).  Its waves share the groups out, and it quantizes the token's
// rows itself: a launch less, and the first weights are on their way meanwhile.  All 16
// columns of the products hold the same token.
constexpr int kOneWaves = 8;

template <class F, bool PAIR>
__global__ __launch_bounds__(64 * kOneWaves) void moe_one_kernel(MoeArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t recs[];
    constexpr int RT = PAIR ? 2 : 1;
    __shared__ float red[kOneWaves][RT][16];
    __shared__ int s_expert[kMoeMaxTopK], s_place[kMoeMaxTopK], s_n;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int g = lane >> 4, r16 = lane & 15;
    const int row0 = 16 * (int)blockIdx.x;
    const size_t pair0 = PAIR ? (size_t)blockIdx.y : (size_t)blockIdx.y * a.top_k;

    // the experts that there are
    int n_seg;
    if (PAIR) {
        const int e = a.ids[pair0];
        if (threadIdx.x == 0) s_expert[0] = e;
        n_seg = e >= 0 ? 1 : 0;
        __syncthreads();
    } else {
        if (wave == 0) {
            const int e = lane < a.top_k ? a.ids[pair0 + lane] : -1;
            const unsigned long long some = __ballot(e >= 0);
            const int at = __popcll(some & ((1ull << lane) - 1ull));
            if (e >= 0) {
                s_expert[at] = e;
                s_place[at] = lane;
            }
            if (lane == 0) s_n = __popcll(some);
        }
        __syncthreads();
        n_seg = s_n;
    }
    const int units = n_seg * a.groups;
    const int u0 = units * wave / kOneWaves, u1 = units * (wave + 1) / kOneWaves;
    const size_t row = (size_t)min(row0 + r16, a.rows - 1) * a.row_bytes;
    const auto load = [&](typename F::W (&w)[RT], int u) {
        const int seg = u / a.groups;
        const size_t at = (size_t)s_expert[seg] * a.expert_bytes + row;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) F::load_w(w[rt], a.w[rt] + at, u - seg * a.groups, a.nblk, g);
    };
    typename F::W w[RT];
    if (u0 < u1) load(w, u0);
    // the token's rows
    const int parts = moe_pack_parts<F::kK>(a.n);
    for (int p = threadIdx.x; p < n_seg * parts; p += 64 * kOneWaves) {
        const int seg = p / parts;
        const size_t from = PAIR ? pair0 / a.top_k : pair0 + s_place[seg];
        moe_pack_part<F::kK>(a.x + from * a.n, a.n, p - seg * parts, recs + (size_t)seg * a.groups * kMoeRec);
    }
    __syncthreads();
    float acc[RT][4] = {};
    for (int u = u0; u < u1; ++u) {
        typename F::W next[RT];
        load(next, min(u + 1, u1 - 1));
        typename F::X x;
        moe_load_x<F>(x, recs + (size_t)u * kMoeRec, g);
        // (down: each group's sum with its expert's weight at once.  A sum kept over an
        // expert's groups needs a branch right behind the products, and the compiler, where a
        // short block lies between, leaves out the wait that their results need)
        const float f = PAIR ? 1.0f : a.weights[pair0 + s_place[u / a.groups]];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            typename F::Op op;
            F::decode(op, w[rt], g);
            MoeScales<F> s;
            s.from(op, g);
            float part[4] = {};
            s.dot(PAIR ? acc[rt] : part, op, x);
            if (!PAIR)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[rt][r] = fmaf(f, part[r], acc[rt][r]);
            w[rt] = next[rt];
        }
    }
    if (r16 == 0)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int r = 0; r < 4; ++r) red[wave][rt][4 * g + r] = acc[rt][r];
    __syncthreads();
    const int o = row0 + (int)threadIdx.x;
    if (threadIdx.x >= 16 || o >= a.rows) return;
    float v[RT] = {};
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int k = 0; k < kOneWaves; ++k) v[rt] += red[k][rt][threadIdx.x];
    if (PAIR) {
        const size_t b = (size_t)max(s_expert[0], 0) * a.rows + o;
        if (a.bias[0] != nullptr) v[0] += a.bias[0][b];
        if (a.bias[1] != nullptr) v[RT - 1] += a.bias[1][b];
        a.out[pair0 * a.rows + o] = n_seg == 0 ? 0.0f : moe_act(v[0], a.activation) * v[RT - 1];
    } else {
        if (a.bias[0] != nullptr)
            for (int j = 0; j < n_seg; ++j)
                v[0] = fmaf(a.weights[pair0 + s_place[j]], a.bias[0][(size_t)s_expert[j] * a.rows + o], v[0]);
        const size_t at = (size_t)blockIdx.y * a.rows + o;
        a.out[at] = a.residual != nullptr ? a.residual[at] + v[0] : v[0];
    }
}

// ------------------------------------------------------------------ few tokens an expert
//
// A workgroup takes 16 rows (gate and up: of each; down: 32) for a tile of up to 16
// TT pairs of one expert; its waves share the groups out, weights straight into
// registers a group ahead, tokens' records from L2, and add their sums in LDS in wave
// order.
constexpr int kFewWaves = 8;

// Rows o .. o + 3 of a pair.
__device__ __forceinline__ void store_rows(float *out, int rows, size_t pair, int o, const float (&v)[4]) {
    float *p = out + pair * rows + o;
    if ((rows & 3) == 0) {
        if (o < rows) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (o + r < rows) p[r] = v[r];
}

// A lane's four rows of a pair from the sums: gate and up to act, down to the pair's part.
template <bool PAIR>
__device__ __forceinline__ void moe_finish(const MoeArgs &a, int e, size_t pair, int o, float (&v)[4], const float (&u)[4]) {
    const size_t b = (size_t)e * a.rows + o;
    float y[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const bool in = o + r < a.rows;
        if (a.bias[0] != nullptr && in) v[r] = a.bias[0][b + r] + v[r];
        if (PAIR) {
            const float up = a.bias[1] != nullptr && in ? a.bias[1][b + r] + u[r] : u[r];
            y[r] = moe_act(v[r], a.activation) * up;
        } else {
            y[r] = a.weights[pair] * v[r];
        }
    }
    store_rows(a.out, a.rows, pair, o, y);
}

template <class F, bool PAIR, int TT>
__global__ __launch_bounds__(64 * kFewWaves) void moe_few_kernel(MoeArgs a) {
    __shared__ float4 red[kFewWaves][2 * TT][64];
    const int n_row = (a.rows + (PAIR ? 15 : 31)) / (PAIR ? 16 : 32);
    const int slot = (int)(blockIdx.x / (unsigned)n_row);
    const MoeTile tile = a.tiles[slot];
    if (tile.count == 0) return;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int g = lane >> 4, r16 = lane & 15;
    const int row0 = (PAIR ? 16 : 32) * ((int)blockIdx.x - slot * n_row);
    const uint8_t *wrow[2];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
        wrow[rt] = a.w[PAIR ? rt : 0] + (size_t)tile.expert * a.expert_bytes +
                   (size_t)min(row0 + (PAIR ? 0 : 16 * rt) + r16, a.rows - 1) * a.row_bytes;
    const uint8_t *rec[TT];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
        const int pair = a.order[tile.start + min(16 * tt + r16, tile.count - 1)];
        rec[tt] = a.pack + (size_t)(PAIR ? pair / a.top_k : pair) * a.groups * kMoeRec;
    }
    const int u0 = a.groups * wave / kFewWaves, u1 = a.groups * (wave + 1) / kFewWaves;
    float acc[2][TT][4] = {};
    if (u0 < u1) {
        typename F::W w[2];
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) F::load_w(w[rt], wrow[rt], u0, a.nblk, g);
        for (int u = u0; u < u1; ++u) {
            typename F::W next[2];
            typename F::X x[TT];
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) moe_load_x<F>(x[tt], rec[tt] + (size_t)u * kMoeRec, g);
#pragma unroll
            for (int rt = 0; rt < 2; ++rt) F::load_w(next[rt], wrow[rt], min(u + 1, u1 - 1), a.nblk, g);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int rt = 0; rt < 2; ++rt) {
                typename F::Op op;
                F::decode(op, w[rt], g);
                MoeScales<F> s;
                s.from(op, g);
#pragma unroll
                for (int tt = 0; tt < TT; ++tt)
                    if (16 * tt < tile.count) s.dot(acc[rt][tt], op, x[tt]);
                w[rt] = next[rt];
            }
        }
    }
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
            red[wave][rt * TT + tt][lane] = make_float4(acc[rt][tt][0], acc[rt][tt][1], acc[rt][tt][2], acc[rt][tt][3]);
    __syncthreads();
    const auto total = [&](int i, int l, float (&v)[4]) {
        v[0] = v[1] = v[2] = v[3] = 0.0f;
#pragma unroll
        for (int k = 0; k < kFewWaves; ++k) {
            const float4 s = red[k][i][l];
            v[0] += s.x, v[1] += s.y, v[2] += s.z, v[3] += s.w;
        }
    };
    for (int i = threadIdx.x; i < (PAIR ? 1 : 2) * TT * 64; i += 64 * kFewWaves) {
        const int l = i & 63, ti = i >> 6, tt = ti % TT, rt = ti / TT;
        const int at = 16 * tt + (l & 15), o = row0 + 16 * rt + 4 * (l >> 4);
        if (at >= tile.count || o >= a.rows) continue;
        float v[4], u[4] = {};
        total(ti, l, v);
        if (PAIR) total(TT + tt, l, u);
        moe_finish<PAIR>(a, tile.expert, (size_t)a.order[tile.start + at], o, v, u);
    }
}

// ------------------------------------------------------------------ a token's parts

// out[t] = [residual[t] +] the parts of its places with an expert, in their order; a
// thread takes 4 rows (VEC) or one.
template <bool VEC>
__global__ __launch_bounds__(256) void moe_join_kernel(const float *__restrict__ part, const int32_t *__restrict__ ids,
                                                       const float *residual, float *out, int m, int top_k, int rows) {
    const int each = VEC ? 4 : 1, per = rows / each;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (size_t)m * per) return;
    const size_t t = i / per;
    const int o = (int)(i - t * per) * each;
    float s[4] = {};
    for (int j = 0; j < top_k; ++j) {
        const size_t pair = t * top_k + j;
        if (ids[pair] < 0) continue;
        const float *p = part + pair * rows + o;
        if (VEC) {
            const float4 v = *reinterpret_cast<const float4 *>(p);
            s[0] += v.x, s[1] += v.y, s[2] += v.z, s[3] += v.w;
        } else {
            s[0] += *p;
        }
    }
    const size_t at = t * rows + o;
    if (residual != nullptr)
#pragma unroll
        for (int r = 0; r < each; ++r) s[r] = residual[at + r] + s[r];
    if (VEC)
        *reinterpret_cast<float4 *>(out + at) = make_float4(s[0], s[1], s[2], s[3]);
    else
        out[at] = s[0];
}

// ------------------------------------------------------------------ launches

namespace {

// LDS of a workgroup of one token that leaves room for two on a CU.
constexpr size_t kOneLds = 60 * 1024;

// Whether a routing's products take a workgroup a token (gate and up: a pair) without sorting the pairs.
bool moe_one(long long pairs) {
    static const int most = tuning_knob("EXQ_MOE_ONE", 16);
    return pairs <= most;
}

// Places a tile of sorted pairs.
int moe_tile(long long pairs, int n_experts) {
    static const int knob = tuning_knob("EXQ_MOE_TILE", 0);
    if (knob != 0) return knob;
    return pairs <= 12LL * n_experts ? 16 : 32;
}

template <class F, bool PAIR>
void moe_pack(const MoeArgs &a, int rows, hipStream_t st) {
    const dim3 grid((unsigned)rows, (unsigned)((moe_pack_parts<F::kK>(a.n) + 255) / 256));
    hipLaunchKernelGGL((moe_pack_kernel<F::kK, PAIR>), grid, dim3(256), 0, st, a);
}

template <class F>
bool moe_run(const edgexpu_hip_moe *p, MoeArgs &a, bool pair, hipStream_t st, const char *what) {
    const long long pairs = (long long)p->pairs();
    if (p->tile == 0) {
        const size_t lds = (size_t)(pair ? 1 : p->top_k) * a.groups * kMoeRec;
        const dim3 grid((unsigned)((a.rows + 15) / 16), (unsigned)(pair ? pairs : p->m));
        if (pair)
            hipLaunchKernelGGL((moe_one_kernel<F, true>), grid, dim3(64 * kOneWaves), lds, st, a);
        else
            hipLaunchKernelGGL((moe_one_kernel<F, false>), grid, dim3(64 * kOneWaves), lds, st, a);
        return lib_hip(hipGetLastError(), what);
    }
    if (pair)
        moe_pack<F, true>(a, p->m, st);
    else
        moe_pack<F, false>(a, (int)pairs, st);
    if (!lib_hip(hipGetLastError(), what)) return false;
    float *out = a.out;
    if (!pair) a.out = p->part;
    const int each = pair ? 16 : 32;
    // (a slot and 16 rows or more a workgroup: what the pairs' rows take in device memory keeps that below 2^31)
    const dim3 grid((unsigned)((a.rows + each - 1) / each) * (unsigned)moe_slots(pairs, p->n_experts, p->tile));
#define MOE_FEW(TT)                                                                                        \
    if (pair)                                                                                              \
        hipLaunchKernelGGL((moe_few_kernel<F, true, TT>), grid, dim3(64 * kFewWaves), 0, st, a);           \
    else                                                                                                   \
        hipLaunchKernelGGL((moe_few_kernel<F, false, TT>), grid, dim3(64 * kFewWaves), 0, st, a);
    if (p->tile == 16) {
        MOE_FEW(1)
    } else {
        MOE_FEW(2)
    }
#undef MOE_FEW
    if (!lib_hip(hipGetLastError(), what)) return false;
    if (pair) return true;
    const bool vec = (a.rows & 3) == 0;
    const unsigned blocks = (unsigned)(((size_t)p->m * (vec ? a.rows / 4 : a.rows) + 255) / 256);
    if (vec)
        hipLaunchKernelGGL(moe_join_kernel<true>, dim3(blocks), dim3(256), 0, st, p->part, a.ids, a.residual, out, p->m,
                           p->top_k, a.rows);
    else
        hipLaunchKernelGGL(moe_join_kernel<false>, dim3(blocks), dim3(256), 0, st, p->part, a.ids, a.residual, out,
                           p->m, p->top_k, a.rows);
    return lib_hip(hipGetLastError(), what);
}

bool moe_product(const edgexpu_hip_moe *p, MoeArgs &a, uint32_t type, bool pair, hipStream_t st, const char *what) {
    switch ((int)type) {
        case kTypeQ4_0: return moe_run<MoeQ40>(p, a, pair, st, what);
        case kTypeQ5_0: return moe_run<MoeQ50>(p, a, pair, st, what);
        case kTypeQ8_0: return moe_run<MoeQ80>(p, a, pair, st, what);
        case kTypeQ4_K: return moe_run<MoeQ4K>(p, a, pair, st, what);
        case kTypeQ5_K: return moe_run<MoeQ5K>(p, a, pair, st, what);
        default: return moe_run<MoeQ6K>(p, a, pair, st, what);
    }
}

// Sorts the pairs of a routing of m tokens where the products need it.
bool moe_plan(edgexpu_hip_moe *p, int m, hipStream_t st, const char *what) {
    const long long pairs = (long long)m * p->top_k;
    const size_t one_lds = (size_t)std::max(moe_groups(p->n_embd), p->top_k * moe_groups(p->n_ff)) * kMoeRec;
    int tile = 0;
    if (m > 0 && (!moe_one(pairs) || one_lds > kOneLds)) {
        tile = moe_tile(pairs, p->n_experts);
        if (!lib_hip(launch_moe_sort(p->ids, (int)pairs, p->n_experts, tile, p->order, p->tiles, st), what)) return false;
    }
    p->tile = tile;
    p->m = m;
    return true;
}

// The checks that the products share.
bool moe_check(const edgexpu_hip_moe *p, const void *w0, const void *w1, uint32_t type, int K, const void *in,
               const void *out, const char *what) {
    if (p == nullptr || p->m < 0) {
        lib_error(-2, "%s: %s", what, p == nullptr ? "null plan" : "the plan has no routing yet");
        return false;
    }
    if (!q8_0_family((int)type) && !k_family((int)type)) {
        lib_error(-3, "%s: GGUF type %u is not supported for experts (Q4_0, Q5_0, Q8_0, Q4_K, Q5_K, Q6_K)", what, type);
        return false;
    }
    const int unit = k_family((int)type) ? kQKK : kQK8_0;
    if (K % unit != 0) {
        lib_error(-2, "%s: rows of %d elements are not whole blocks of type %u", what, K, type);
        return false;
    }
    if (p->m == 0) return true;
    if (w0 == nullptr || w1 == nullptr || in == nullptr || out == nullptr) {
        lib_error(-2, "%s: null buffer", what);
        return false;
    }
    if ((((uintptr_t)w0 | (uintptr_t)w1 | (uintptr_t)in | (uintptr_t)out) & 15u) != 0) {
        lib_error(-2, "%s: weights and activations must be 16-byte aligned", what);
        return false;
    }
    return true;
}

size_t block_bytes(uint32_t type) {
    switch ((int)type) {
        case kTypeQ4_0: return kBytesQ4_0;
        case kTypeQ5_0: return kBytesQ5_0;
        case kTypeQ8_0: return kBytesQ8_0;
        case kTypeQ4_K: return kBytesQ4_K;
        case kTypeQ5_K: return kBytesQ5_K;
        default: return kBytesQ6_K;
    }
}

MoeArgs moe_args(const edgexpu_hip_moe *p, uint32_t type, int rows, int n) {
    MoeArgs a = {};
    a.ids = p->ids;
    a.weights = p->weights;
    a.order = p->order;
    a.tiles = p->tiles;
    a.pack = p->pack;
    a.n = n;
    a.nblk = n / (k_family((int)type) ? kQKK : kQK8_0);
    a.groups = moe_groups(n);
    a.row_bytes = a.nblk * block_bytes(type);
    a.expert_bytes = a.row_bytes * (size_t)rows;
    a.m = p->m;
    a.top_k = p->top_k;
    a.rows = rows;
    return a;
}

}  // namespace

}  // namespace exq

using namespace exq;

extern "C" {

edgexpu_hip_moe *edgexpu_hip_moe_create(int n_experts, int top_k, int max_tokens, int n_embd, int n_ff) {
    if (n_experts <= 0 || n_experts > kMoeMaxExperts || top_k <= 0 || top_k > n_experts || top_k > kMoeMaxTopK ||
        max_tokens <= 0 || (long long)max_tokens * top_k > (1 << 22) || n_embd <= 0 || n_embd > (1 << 20) ||
        n_ff <= 0 || n_ff > (1 << 20)) {
        lib_error(-2, "moe_create: %d of %d experts (at most %d of %d), %d tokens or rows of %d and %d out of range", top_k,
                  n_experts, kMoeMaxTopK, kMoeMaxExperts, max_tokens, n_embd, n_ff);
        return nullptr;
    }
    if (!lib_ready("moe_create")) return nullptr;
    edgexpu_hip_moe *p = new (std::nothrow) edgexpu_hip_moe();
    if (p == nullptr) {
        lib_error(-5, "moe_create: out of host memory");
        return nullptr;
    }
    p->n_experts = n_experts;
    p->top_k = top_k;
    p->max_tokens = max_tokens;
    p->n_embd = n_embd;
    p->n_ff = n_ff;
    const size_t pairs = (size_t)max_tokens * top_k;
    const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t sizes[6] = {4 * pairs, 4 * pairs, 4 * pairs, sizeof(MoeTile) * moe_slots(pairs, n_experts, 16),
                             kMoeRec * std::max((size_t)moe_groups(n_embd) * max_tokens, (size_t)moe_groups(n_ff) * pairs),
                             4 * pairs * n_embd};
    size_t total = 0, at[6];
    for (int i = 0; i < 6; ++i) {
        at[i] = total;
        total += up(sizes[i]);
    }
    if (!lib_hip(hipMalloc((void **)&p->mem, total), "moe_create: hipMalloc")) {
        delete p;
        return nullptr;
    }
    p->ids = (int32_t *)p->mem;
    p->weights = (float *)(p->mem + at[1]);
    p->order = (int32_t *)(p->mem + at[2]);
    p->tiles = (MoeTile *)(p->mem + at[3]);
    p->pack = p->mem + at[4];
    p->part = (float *)(p->mem + at[5]);
    return p;
}

void edgexpu_hip_moe_destroy(edgexpu_hip_moe *p) {
    if (p == nullptr) return;
    (void)hipDeviceSynchronize();
    (void)hipFree(p->mem);
    delete p;
}

int edgexpu_hip_moe_tokens(const edgexpu_hip_moe *p) { return p != nullptr && p->m > 0 ? p->m : 0; }

int edgexpu_hip_moe_route_dev(edgexpu_hip_moe *p, int32_t *ids, float *weights, const float *scores, int m, int score,
                              const float *bias, int n_groups, int top_groups, int group_best, int normalise,
                              double scale, void *stream) {
    if (p == nullptr || m < 0 || m > p->max_tokens || (m > 0 && scores == nullptr)) {
        lib_error(-2, "moe_route: null plan or scores, or %d tokens (at most %d)", m, p != nullptr ? p->max_tokens : 0);
        return 0;
    }
    if ((score != EDGEXPU_HIP_MOE_SOFTMAX && score != EDGEXPU_HIP_MOE_SIGMOID) || n_groups < 1 ||
        n_groups > kMoeMaxGroups || p->n_experts % n_groups != 0 || top_groups < 1 || top_groups > n_groups ||
        group_best < 1 || group_best > 2 || !std::isfinite(scale)) {
        lib_error(-2, "moe_route: score %d, best %d of groups (%d of %d, %d experts) or scale %g out of range", score,
                  group_best, top_groups, n_groups, p->n_experts, scale);
        return 0;
    }
    if (!lib_ready("moe_route")) return 0;
    if (m > 0) {
        RouteArgs a = {};
        a.scores = scores;
        a.bias = bias;
        a.ids = p->ids;
        a.ids_out = ids;
        a.weights = p->weights;
        a.weights_out = weights;
        a.m = m;
        a.n_experts = p->n_experts;
        a.top_k = p->top_k;
        a.sigmoid = score == EDGEXPU_HIP_MOE_SIGMOID;
        a.n_groups = n_groups;
        a.top_groups = top_groups;
        a.group_best = group_best;
        a.normalise = normalise != 0;
        a.scale = scale;
        if (!lib_hip(launch_moe_route(a, (hipStream_t)stream), "moe_route")) return 0;
    }
    return moe_plan(p, m, (hipStream_t)stream, "moe_route") ? 1 : 0;
}

int edgexpu_hip_moe_assign_dev(edgexpu_hip_moe *p, const int32_t *ids, const float *weights, int m, void *stream) {
    if (p == nullptr || m < 0 || m > p->max_tokens || (m > 0 && (ids == nullptr || weights == nullptr))) {
        lib_error(-2, "moe_assign: null plan, ids or weights, or %d tokens (at most %d)", m,
                  p != nullptr ? p->max_tokens : 0);
        return 0;
    }
    if (!lib_ready("moe_assign")) return 0;
    if (m > 0 && !lib_hip(launch_moe_assign(ids, weights, p->ids, p->weights, m * p->top_k, p->n_experts,
                                            (hipStream_t)stream), "moe_assign"))
        return 0;
    return moe_plan(p, m, (hipStream_t)stream, "moe_assign") ? 1 : 0;
}

int edgexpu_hip_moe_gate_up_dev(float *act, const float *x, edgexpu_hip_moe *p, const void *w_gate, const void *w_up,
                                uint32_t type, const float *b_gate, const float *b_up, int activation, void *stream) {
    const char *what = "moe_gate_up";
    if (activation != EDGEXPU_HIP_MOE_SILU && activation != EDGEXPU_HIP_MOE_GELU) {
        lib_error(-2, "%s: unknown activation %d", what, activation);
        return 0;
    }
    if (!moe_check(p, w_gate, w_up, type, p != nullptr ? p->n_embd : 0, x, act, what) || !lib_ready(what)) return 0;
    if (p->m == 0) return 1;
    MoeArgs a = moe_args(p, type, p->n_ff, p->n_embd);
    a.w[0] = (const uint8_t *)w_gate;
    a.w[1] = (const uint8_t *)w_up;
    a.bias[0] = b_gate;
    a.bias[1] = b_up;
    a.activation = activation;
    a.x = x;
    a.out = act;
    return moe_product(p, a, type, true, (hipStream_t)stream, what) ? 1 : 0;
}

int edgexpu_hip_moe_down_dev(float *out, const float *act, edgexpu_hip_moe *p, const void *w_down, uint32_t type,
                             const float *bias, const float *residual, void *stream) {
    const char *what = "moe_down";
    if (!moe_check(p, w_down, w_down, type, p != nullptr ? p->n_ff : 0, act, out, what) || !lib_ready(what)) return 0;
    if (p->m == 0) return 1;
    MoeArgs a = moe_args(p, type, p->n_embd, p->n_ff);
    a.w[0] = (const uint8_t *)w_down;
    a.bias[0] = bias;
    a.residual = residual;
    a.x = act;
    a.out = out;
    return moe_product(p, a, type, false, (hipStream_t)stream, what) ? 1 : 0;
}

}  // extern "C"
