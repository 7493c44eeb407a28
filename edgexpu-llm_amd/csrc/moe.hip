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
constexpr float kNan = __builtin_nanf("");
__device__ __forceinline__ float moe_act(float v, int activation) {
    return activation == EDGEXPU_HIP_MOE_GELU ? gelu_f32(v) : silu_f32(v);
}

struct MoeArgs {
    const int32_t *routed;    // holds m, or the plan's routing is not of these tokens: NaN, and nothing of it is read
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
// tokens, and the places of a token that have no expert get zeros in `out` by the way
// (without a routing of these tokens all of them NaN).
template <bool K, bool ACT>
__global__ __launch_bounds__(256) void moe_pack_kernel(MoeArgs a) {
    const size_t row = blockIdx.x;
    const int part = (int)blockIdx.y * 256 + (int)threadIdx.x;
    if (part < moe_pack_parts<K>(a.n))
        moe_pack_part<K>(a.x + row * a.n, a.n, part, a.pack + row * a.groups * kMoeRec);
    if (ACT && blockIdx.y == 0) {
        const bool routed = *a.routed == a.m;
        for (int j = 0; j < a.top_k; ++j) {
            const size_t pair = row * a.top_k + j;
            if (!routed || a.ids[pair] < 0)
                for (int i = threadIdx.x; i < a.rows; i += 256) a.out[pair * a.rows + i] = routed ? 0.0f : kNan;
        }
    }
}

// ------------------------------------------------------------------ one token
//
// A workgroup takes 16 rows (gate and up: of each) for one token: of one of its
// experts (gate and up), or of all of them, whose weighted sum then needs no second
// launch (down).  Its waves share the groups out, and it quantizes the token's
// rows itself: a launch less, and the first weights are on their way meanwhile.  All 16
// columns of the products hold the same token.
// What bounds it: for a token a chain (arguments 0.7 us, choice 0.9, weights 2, products, sums
// 1.2): 8 of 128 experts of 768 x 2560, Q4_K, gate and up 7.4 us; down of 2560 x 768, Q6_K, 10.3, the decoding of three
// groups a wave; for more pairs the memory: 3 tokens of 14336 x 4096 79 us, 3.9 TB/s.  At most
// 128 registers, so that two workgroups fit a CU (162: gate and up 10.0 us); 16 waves, down 12.7.
constexpr int kOneWaves = 8;

template <class F, bool PAIR>
__global__ __launch_bounds__(64 * kOneWaves, 4) void moe_one_kernel(MoeArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t recs[];
    // gate and up: half the waves each
    constexpr int kSets = PAIR ? 2 : 1, kShare = kOneWaves / kSets;
    // groups whose weights are on their way at once: a wave of a single token mostly has no more
    constexpr int kAhead = F::kK ? 2 : 1;
    __shared__ __attribute__((aligned(16))) float red[kOneWaves][16];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int g = lane >> 4, r16 = lane & 15;
    const int row0 = 16 * (int)blockIdx.x;
    const size_t pair0 = PAIR ? (size_t)blockIdx.y : (size_t)blockIdx.y * a.top_k;

    // The token's rows need nothing from its experts: the first are read before them.
    const int parts = moe_pack_parts<F::kK>(a.n), all = PAIR ? parts : a.top_k * parts;
    const float *x = a.x + (PAIR ? pair0 / a.top_k : pair0) * a.n;
    const auto read = [&](float (&v)[F::kK ? 16 : 8], int p) {
        const int place = PAIR ? 0 : p / parts;
        moe_read_part<F::kK>(v, x + (size_t)place * a.n, a.n, p - place * parts);
    };
    float first[F::kK ? 16 : 8];
    if ((int)threadIdx.x < all) read(first, threadIdx.x);

    // Lane j's expert, place and weight: the j-th that there is (every wave for itself).
    const int own = PAIR ? 0 : lane;
    const bool routed = *a.routed == a.m;
    int expert = own < (PAIR ? 1 : a.top_k) ? a.ids[pair0 + own] : -1, place = own, n_seg;
    if (!routed) expert = -1;
    float weight = 1.0f;
    if (PAIR) {
        n_seg = expert >= 0 ? 1 : 0;
    } else {
        weight = lane < a.top_k ? a.weights[pair0 + lane] : 0.0f;
        const unsigned long long some = __ballot(expert >= 0), below = (1ull << lane) - 1ull;
        n_seg = __popcll(some);
        const int at = 4 * (expert >= 0 ? __popcll(some & below) : n_seg + __popcll(~some & below));
        expert = __builtin_amdgcn_ds_permute(at, expert);
        place = __builtin_amdgcn_ds_permute(at, place);
        weight = __int_as_float(__builtin_amdgcn_ds_permute(at, __float_as_int(weight)));
    }
    const auto nth = [](int v, int seg) { return PAIR ? v : __builtin_amdgcn_readlane(v, seg); };
    const int units = n_seg * a.groups;
    const int part = wave & (kShare - 1), u0 = units * part / kShare, u1 = units * (part + 1) / kShare;
    const uint8_t *rows = a.w[wave / kShare] + (size_t)min(row0 + r16, a.rows - 1) * a.row_bytes;
    const auto load = [&](typename F::W &w, int u) {
        if (u >= u1) return;
        const int seg = PAIR ? 0 : u / a.groups;
        F::load_w(w, rows + (size_t)nth(expert, seg) * a.expert_bytes, u - seg * a.groups, a.nblk, g);
    };
    typename F::W w[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) load(w[k], u0 + k);
    if ((int)threadIdx.x < all) moe_put_part<F::kK>(first, threadIdx.x, recs);
    for (int p = threadIdx.x + 64 * kOneWaves; p < all; p += 64 * kOneWaves) {
        read(first, p);
        moe_put_part<F::kK>(first, p, recs);
    }
    __syncthreads();
    float acc[4] = {};
    for (int base = u0; base < u1; base += kAhead)
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int u = base + k;
            if (u >= u1) break;
            const int seg = PAIR ? 0 : u / a.groups;
            typename F::Op op;
            F::decode(op, w[k], g);
            moe_hold_op(op);
            __builtin_amdgcn_sched_barrier(0);
            load(w[k], u + kAhead);
            typename F::X x;
            moe_load_x<F>(x, recs + ((size_t)nth(place, seg) * a.groups + (u - seg * a.groups)) * kMoeRec, g);
            MoeScales<F> s;
            s.from(op, g);
            // (down: each group's sum with its expert's weight at once.  A sum kept over an
            // expert's groups needs a branch right behind the products, and the compiler, where a
            // short block lies between, leaves out the wait that their results need)
            const float f = __int_as_float(nth(__float_as_int(weight), seg));
            float one[4] = {};
            s.dot(PAIR ? acc : one, op, x);
            if (!PAIR)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[r] = fmaf(f, one[r], acc[r]);
        }
    if (r16 == 0) *reinterpret_cast<float4 *>(&red[wave][4 * g]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    __syncthreads();
    const int o = row0 + (int)threadIdx.x;
    if (threadIdx.x >= 16 || o >= a.rows) return;
    float v[kSets] = {};
#pragma unroll
    for (int k = 0; k < kOneWaves; ++k) v[k / kShare] += red[k][threadIdx.x];
    if (PAIR) {
        const size_t b = (size_t)max(expert, 0) * a.rows + o;
        if (a.bias[0] != nullptr) v[0] += a.bias[0][b];
        if (a.bias[1] != nullptr) v[kSets - 1] += a.bias[1][b];
        const float y = n_seg == 0 ? 0.0f : moe_act(v[0], a.activation) * v[kSets - 1];
        a.out[pair0 * a.rows + o] = routed ? y : kNan;
    } else {
        if (a.bias[0] != nullptr)
            for (int j = 0; j < n_seg; ++j)
                v[0] = fmaf(__int_as_float(nth(__float_as_int(weight), j)), a.bias[0][(size_t)nth(expert, j) * a.rows + o], v[0]);
        const size_t at = (size_t)blockIdx.y * a.rows + o;
        const float y = a.residual != nullptr ? a.residual[at] + v[0] : v[0];
        a.out[at] = routed ? y : kNan;
    }
}

// ------------------------------------------------------------------ tiles of pairs
//
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

// One LDS DMA: lane l's 16 bytes at src land at LDS address lds + 16 l.  Its wait is
// wait_loads(): the compiler knows of neither, and its own waits for the weights
// only ever wait for more.  (M0, which the compiler reserves, is put back.)
__device__ __forceinline__ void dma16(uint32_t lds, const uint8_t *src) {
    uint32_t saved;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %1\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %2, off\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "s"(lds), "v"(src)
        : "memory");
}
template <int N>
__device__ __forceinline__ void wait_loads() {  // at most N loads or DMAs still on their way
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
__device__ __forceinline__ uint32_t lds_addr(const void *p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)p;
}

// A workgroup of 4 waves takes a tile's pairs, up to T = 16 TT of one expert, against a
// block of weight rows: two tiles of 16 rows a wave (gate and up: one of each), or with
// KS > 1 KS waves share two tiles' groups out.  Weights go straight from memory into
// registers, each row read by one wave, DEEP groups ahead of their products; the tokens'
// records, which all waves read, come through LDS by DMA, CH groups of T tokens a
// buffer, two buffers.  A step takes one of its row tiles after the other, so that
// only one's decoded rows are in registers (both at once read each record once, but with a
// third more registers and 2 waves a SIMD for 3: 512 tokens 109 us so, 103 one by one).
// What bounds it: memory where tiles are few (12 tokens of 8 experts, 4096 rows of 14336, Q4_K, 54 us, 4.7 TB/s); with
// many pairs an expert vector instructions, to decode a row tile's group 110 (Q4_K) to 450 (Q6_K), and 20 for 16 pairs'
// scales (4096 tokens of 128 experts, 768 rows of 2560 twice, Q4_K, 397 us, 650 TFLOP/s: they issue in 70 % of the
// cycles); between the two how far loads and products overlap (512 tokens 100 us: bytes 61, vector instructions 44,
// matrix products 18, waves wait 40 % of their time).
__host__ __device__ constexpr int tile_chunk(int TT) { return TT == 2 ? 2 : 1; }
__host__ __device__ constexpr int tile_lds(int TT) { return 2 * tile_chunk(TT) * 16 * TT * kMoeRec; }
constexpr int kTileWaves = 4;
// Row blocks in a row on a chiplet: enough that they share a tile's records in its L2, few enough that every
// chiplet has its part where slots are few or empty (16 tokens of 8 experts, 14336 rows of 4096: 124 us, with an eighth of the
// slots a chiplet 219; 4096 tokens of 128 experts, 2560 rows of 768: 449 and 469, one by one 468).
constexpr int kRun = 4;
// Groups of weights ahead: two where a step's products are too short to hide a load behind.  Not for
// formats whose decoding is long: it is then what hides the load, and a second copy of it only costs
// registers and instruction fetches (Q6_K, 64 tokens of 128 experts, 2560 rows of 768: 82 us with one, 89 with two).
template <class F>
constexpr int tile_deep(int TT) { return !F::kLong && TT <= 2 ? 2 : 1; }

// Sums made where they stand: left to the compiler, all tiles' integer sums wait in
// registers for the end of a step.
__device__ __forceinline__ void pin(float (&v)[4]) {
    asm volatile("" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]));
}

template <class F, bool PAIR, int TT, int DEEP>
__global__ __launch_bounds__(64 * kTileWaves, 2) void moe_tile_kernel(MoeArgs a, int ks_log, int each, int slots, int n_blk) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ int s_pair[16 * TT];
    constexpr int T = 16 * TT, CH = tile_chunk(TT), kBuf = CH * T * kMoeRec;
    constexpr int kDma = kBuf / 1024, kEach = (kDma + kTileWaves - 1) / kTileWaves;
    static_assert(kBuf % 1024 == 0, "whole DMAs");
    // Workgroup b runs on chiplet b % 8: the row blocks of all slots, one slot after the other, go to
    // the chiplets in runs of kRun.
    const int turn = (int)(blockIdx.x >> 3), f = ((turn / kRun << 3) + (int)(blockIdx.x & 7u)) * kRun + turn % kRun;
    const int slot = f / n_blk, blk = f - slot * n_blk;
    if (slot >= slots) return;
    const MoeTile tile = a.tiles[slot];
    if (*a.routed != a.m) return;  // (the tiles are another routing's)
    if (tile.rest == 0 || tile.index % each != 0) return;  // (this kernel's tile is `each` of the sort's)
    const int pairs = min(tile.rest, T);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int g = lane >> 4, r16 = lane & 15;
    const int KS = 1 << ks_log, ks = wave & (KS - 1);
    constexpr int kRows = PAIR ? 16 : 32;
    const int row0 = kRows * (blk * (kTileWaves >> ks_log) + (wave >> ks_log));
    const int u0 = a.groups * ks >> ks_log, u1 = a.groups * (ks + 1) >> ks_log;
    const int chs = CH >> ks_log;  // groups of a part in a buffer
    const int n_chunk = (((a.groups + KS - 1) >> ks_log) + chs - 1) / chs, n_step = n_chunk * chs;

    if ((int)threadIdx.x < T) s_pair[threadIdx.x] = a.order[tile.start + min((int)threadIdx.x, pairs - 1)];
    __syncthreads();
    // The DMAs' sources, in units of 16 bytes: piece p of a buffer is piece p % 19 of record
    // p / 19, token p / 19 % T's group p / 19 / T: group p / 19 / T / KS of part p / 19 / T % KS.
    uint32_t from[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int p = min(i * kTileWaves + wave, kDma - 1) * 64 + lane;
        const int rec = p / (kMoeRec / 16), c = rec / T;
        const int u = (a.groups * (c & (KS - 1)) >> ks_log) + (c >> ks_log);
        const unsigned pair = (unsigned)s_pair[rec - c * T];
        const unsigned row = PAIR ? pair / (unsigned)a.top_k : pair;
        from[i] = (row * (unsigned)a.groups + u) * (kMoeRec / 16) + (p - rec * (kMoeRec / 16));
    }
    const auto stage = [&](int buf) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int d = i * kTileWaves + wave;
            if (d < kDma) dma16(lds_addr(lds) + buf * kBuf + 1024 * d, a.pack + ((size_t)from[i] << 4));
            from[i] += (unsigned)chs * (kMoeRec / 16);
        }
    };
    const uint8_t *wrow[2];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
        wrow[rt] = a.w[PAIR ? rt : 0] + (size_t)tile.expert * a.expert_bytes +
                   (size_t)min(row0 + (PAIR ? 0 : 16 * rt) + r16, a.rows - 1) * a.row_bytes;
    float acc[2][TT][4] = {};
    typename F::W w[DEEP][2];
    int next = u0;  // the next loads' group; past the end the last one again
    const auto load = [&](typename F::W &wv, int rt) { F::load_w(wv, wrow[rt], max(min(next, u1 - 1), 0), a.nblk, g); };
    stage(0);
#pragma unroll
    for (int k = 0; k < DEEP; ++k) {
        load(w[k][0], 0);
        load(w[k][1], 1);
        ++next;
    }
    // Both row tiles against a buffer's group.  Every step loads, so that the wait for a
    // step's weights counts the same loads on every path.
    const auto step = [&](int v, typename F::W (&wv)[2]) {
        if ((v & (chs - 1)) == 0) {
            // a buffer's DMAs are older than the last step's loads, of which the 16-byte ones
            // (Q4_K: 3 a row tile, the others more) are surely one instruction each
            wait_loads<6>();
            __syncthreads();  // this buffer is whole, and the other one has been read
            if (v + chs < n_step) stage((v / chs + 1) & 1);
        }
        const uint8_t *rec = lds + ((v / chs) & 1) * kBuf + (((v & (chs - 1)) << ks_log) + ks) * (T * kMoeRec) + r16 * kMoeRec;
        const int count = u0 + v < u1 ? pairs : 0;
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
            typename F::Op op;
            MoeScales<F> s;
            F::decode(op, wv[rt], g);
            moe_hold_op(op);
            s.from(op, g);
            __builtin_amdgcn_sched_barrier(0);
            load(wv[rt], rt);
            if (rt == 1) ++next;
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                if (16 * tt >= count) break;
                typename F::X x;
                moe_load_x<F>(x, rec + 16 * tt * kMoeRec, g);
                s.dot(acc[rt][tt], op, x);
                pin(acc[rt][tt]);
            }
        }
    };
    int v = 0;
    const int n_end = ks_log == 0 ? a.groups : n_step;  // (parts may differ by a group, and meet at the same barriers)
    for (; v + DEEP <= n_end; v += DEEP)
#pragma unroll
        for (int k = 0; k < DEEP; ++k) step(v + k, w[k]);
    if (DEEP == 2 && v < n_end) step(v, w[0]);
    if (KS > 1) {  // the parts' sums, in their order
        float4 *red = reinterpret_cast<float4 *>(lds);
        __syncthreads();
        if (ks > 0)
#pragma unroll
            for (int rt = 0; rt < 2; ++rt)
#pragma unroll
                for (int tt = 0; tt < TT; ++tt)
                    red[((wave * 2 + rt) * TT + tt) * 64 + lane] =
                        make_float4(acc[rt][tt][0], acc[rt][tt][1], acc[rt][tt][2], acc[rt][tt][3]);
        __syncthreads();
        if (ks > 0) return;
        for (int k = 1; k < KS; ++k)
#pragma unroll
            for (int rt = 0; rt < 2; ++rt)
#pragma unroll
                for (int tt = 0; tt < TT; ++tt) {
                    const float4 o = red[(((wave + k) * 2 + rt) * TT + tt) * 64 + lane];
                    acc[rt][tt][0] += o.x, acc[rt][tt][1] += o.y, acc[rt][tt][2] += o.z, acc[rt][tt][3] += o.w;
                }
    }
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
        const int at = 16 * tt + r16;
        if (at >= pairs) continue;
        const size_t pair = (size_t)s_pair[at];
        if (PAIR) {
            if (row0 + 4 * g < a.rows)
                moe_finish<true>(a, tile.expert, pair, row0 + 4 * g, acc[0][tt], acc[1][tt]);
        } else {
#pragma unroll
            for (int rt = 0; rt < 2; ++rt)
                if (row0 + 16 * rt + 4 * g < a.rows)
                    moe_finish<false>(a, tile.expert, pair, row0 + 16 * rt + 4 * g, acc[rt][tt], acc[rt][tt]);
        }
    }
}

template <class F, bool PAIR, int TT>
constexpr auto tile_kernel() {
    return moe_tile_kernel<F, PAIR, TT, tile_deep<F>(TT)>;
}

// ------------------------------------------------------------------ a token's parts

// out[t] = [residual[t] +] the parts of its places with an expert, in their order; a
// thread takes 4 rows (VEC) or one.  One pass over the parts: 4096 tokens of 8 x 2560, 81 us, 5.2 TB/s, part of them from the caches.
template <bool VEC>
__global__ __launch_bounds__(256) void moe_join_kernel(const float *__restrict__ part, const int32_t *__restrict__ ids,
                                                       const int32_t *__restrict__ routed, const float *residual,
                                                       float *out, int m, int top_k, int rows) {
    const int each = VEC ? 4 : 1, per = rows / each;
    const bool whole = *routed == m;
    // (a turn, except where the rows are more than a launch's threads may be)
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < (size_t)m * per; i += (size_t)gridDim.x * 256) {
        const size_t t = i / per;
        const int o = (int)(i - t * per) * each;
        float s[4] = {};
        for (int j = 0; whole && j < top_k; ++j) {
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
        if (!whole)
#pragma unroll
            for (int r = 0; r < each; ++r) s[r] = kNan;
        if (VEC)
            *reinterpret_cast<float4 *>(out + at) = make_float4(s[0], s[1], s[2], s[3]);
        else
            out[at] = s[0];
    }
}

// ------------------------------------------------------------------ launches

// Threads of a launch in x, and workgroups of 256: 2^32 and more are taken modulo 2^32.
constexpr size_t kLaunch = (size_t)1 << 31;
constexpr long long kMoeBlocks = (1 << 24) - 32;

// LDS of a workgroup of one token that leaves room for two on a CU.
constexpr size_t kOneLds = 60 * 1024;

// Whether a product takes a workgroup a token (gate and up: a pair) without sorting the pairs: where few experts
// have two tokens, whose weights the tiles read once.  `weights`: an expert's elements in the product.  The tiles' launches
// cost some 20 us, so that up to 8 pairs of smaller experts are faster without them; the larger an expert, the
// fewer pairs (us so and with tiles, Q4_K, the weights from memory; their sort costs 5 besides:
//   128 experts of 768 x 2560, gate and up: 64 pairs 32 and 30, 96 pairs 45 and 38; down (Q6_K): 35 and 38, 53 and 48
//   gate and up, 14336 x 4096: 8 experts, 6 pairs 92 and 90, 8 pairs 119 and 90; 4 experts, 4 pairs 64 and 58, 6 pairs 88 and 58
//   gate and up, 4096 x 4096: 8 experts, 8 pairs 39 and 39; 4 experts, 6 pairs 28 and 24, 8 pairs 37 and 26
//   down, 4096 x 14336: 8 experts, 8 pairs 59 and 65; 4 experts, 6 pairs 46 and 46, 8 pairs 60 and 47).
bool moe_takes_one(long long pairs, int n_experts, long long weights, size_t lds) {
    const int half = n_experts / 2;
    int most = std::max(8, half);
    if (weights >= 1 << 26)
        most = std::min(most, half + 2);
    else if (weights >= 1 << 25)
        most = std::min(most, half + 5);
    return pairs <= most && lds <= kOneLds;
}

// Pairs an expert from which tiles hold 128 of them (0: none do), where a decoded row is worth it (us of gate, up and down
// with 64 and 128, experts of 768 x 2560:
//   Q6_K  50 pairs of each of 128 experts 394 and 369; of 32, 48 pairs 142 and 154, 64 pairs 151 and 143
//   Q5_0  of 128, 64 pairs 781 and 772, 96 pairs 963 and 882; of 32, 64 pairs 253 and 296, 96 pairs 323 and 331
//   Q8_0  of 128, 96 pairs 734 and 721, 128 pairs 886 and 792; of 32, 64 pairs 208 and 237, 192 pairs 346 and 328
//   128 pairs: of 128, Q4_0 820 and 902; of 32, Q4_K 133 and 154, Q5_K 147 and 172).
constexpr int wide_from(int type) {
    return type == kTypeQ6_K ? 50 : type == kTypeQ5_0 ? 96 : type == kTypeQ8_0 ? 128 : 0;
}
bool moe_takes_wide(int type, long long pairs, int n_experts) {
    return wide_from(type) > 0 && pairs >= (long long)wide_from(type) * n_experts;
}

namespace {

// A routing of m tokens in gate and up (`pair`), or in down, whose workgroups hold all of a token's rows.
bool moe_one(const edgexpu_hip_moe *p, int m, bool pair) {
    const size_t records = pair ? moe_groups(p->n_embd) : (size_t)p->top_k * moe_groups(p->n_ff);
    return moe_takes_one((long long)m * p->top_k, p->n_experts, (pair ? 2LL : 1LL) * p->n_embd * p->n_ff,
                         records * kMoeRec);
}

// Places a tile of sorted pairs (us with 32 and 64, 128 experts of 768 x 2560: 8 pairs an expert, gate and up 64 and 71,
// down Q6_K 79 and 90; 16 pairs 83 and 79, 100 and 94).
int moe_tile(long long pairs, int n_experts) {
    return pairs < 16LL * n_experts ? 32 : 64;
}

template <class F, bool PAIR, int TT>
void moe_tiles(const MoeArgs &a, int each, int slots, int ks_log, hipStream_t st) {
    const int rows = (PAIR ? 16 : 32) * (kTileWaves >> ks_log);
    const int n_blk = (a.rows + rows - 1) / rows;
    // (at most kMoeBlocks, up to whole runs: _create's limit for gate and up; down's parts, 4 bytes each, are below 2^37 in
    // the device's memory, which with 512 experts of 2^20 rows is 2^37 / (64 128) + 2^22 workgroups)
    const dim3 grid((unsigned)((slots * n_blk + 8 * kRun - 1) / (8 * kRun)) * 8u * kRun);
    hipLaunchKernelGGL((tile_kernel<F, PAIR, TT>()), grid, dim3(64 * kTileWaves), tile_lds(TT), st, a, ks_log, each,
                       slots, n_blk);
}

template <class F, bool PAIR>
void moe_pack(const MoeArgs &a, int rows, hipStream_t st) {
    const dim3 grid((unsigned)rows, (unsigned)((moe_pack_parts<F::kK>(a.n) + 255) / 256));
    hipLaunchKernelGGL((moe_pack_kernel<F::kK, PAIR>), grid, dim3(256), 0, st, a);
}

template <class F>
bool moe_run(const edgexpu_hip_moe *p, MoeArgs &a, bool pair, hipStream_t st, const char *what) {
    const long long pairs = (long long)p->pairs();
    if (moe_one(p, p->m, pair)) {
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
    const int slots = moe_slots(pairs, p->n_experts, p->tile);
    // two waves share two row tiles' groups where the tiles are too few to fill the chip (12 tokens
    // of 8 experts, 4096 rows of 14336: 256 workgroups 69 us, 512 so 63; where they are enough, 333 tokens of 64
    // experts, 2560 rows of 1024, 75 us and 88 so)
    const long long blocks = (std::min<long long>(p->n_experts, pairs) + pairs / 32) * ((a.rows + 127) / 128);
    const int ks = p->tile == 32 && !pair && blocks < 512 ? 1 : 0;
    const bool wide = moe_takes_wide(F::kType, pairs, p->n_experts);
#define MOE_TILES(TT, EACH)                              \
    if (pair)                                            \
        moe_tiles<F, true, TT>(a, EACH, slots, ks, st);  \
    else                                                 \
        moe_tiles<F, false, TT>(a, EACH, slots, ks, st);
    if (p->tile == 32) {
        MOE_TILES(2, 1)
    } else if (!wide) {
        MOE_TILES(4, 1)
    } else if constexpr (wide_from(F::kType) > 0) {
        MOE_TILES(8, 2)
    }
#undef MOE_TILES
    if (!lib_hip(hipGetLastError(), what)) return false;
    if (pair) return true;
    const bool vec = (a.rows & 3) == 0;
    const unsigned joins = (unsigned)std::min(((size_t)p->m * (vec ? a.rows / 4 : a.rows) + 255) / 256, kLaunch / 256);
    if (vec)
        hipLaunchKernelGGL(moe_join_kernel<true>, dim3(joins), dim3(256), 0, st, p->part, a.ids, a.routed, a.residual,
                           out, p->m, p->top_k, a.rows);
    else
        hipLaunchKernelGGL(moe_join_kernel<false>, dim3(joins), dim3(256), 0, st, p->part, a.ids, a.routed, a.residual,
                           out, p->m, p->top_k, a.rows);
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

// Places a tile of the sorted pairs of a routing of m tokens; 0 where no product needs them sorted.
int moe_sorted(const edgexpu_hip_moe *p, int m) {
    if (m == 0 || (moe_one(p, m, true) && moe_one(p, m, false))) return 0;
    return moe_tile((long long)m * p->top_k, p->n_experts);
}

// Sorts the pairs of a routing of m tokens where the products need it.
bool moe_plan(edgexpu_hip_moe *p, int m, hipStream_t st, const char *what) {
    const int tile = moe_sorted(p, m);
    if (tile != 0 && !lib_hip(launch_moe_sort(p->ids, m * p->top_k, p->n_experts, tile, p->order, p->tiles, p->routed, m,
                                              st), what))
        return false;
    p->tile = tile;
    p->m = m;
    return true;
}

// LDS beyond 64 KiB is asked for once, when a plan is made: nothing of it is left for a captured call.
template <class F>
bool moe_prepare() {
    const void *k[2] = {(const void *)tile_kernel<F, true, 8>(), (const void *)tile_kernel<F, false, 8>()};
    for (const void *f : k)
        if (!lib_hip(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, tile_lds(8)), "moe_create"))
            return false;
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
    a.routed = p->routed;
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
    const size_t pairs = (size_t)max_tokens * top_k;
    const size_t records = std::max((size_t)moe_groups(n_embd) * max_tokens, (size_t)moe_groups(n_ff) * pairs);
    if (records > (size_t)1 << 27) {  // (their places are counted in 32 bits, 16 bytes a unit)
        lib_error(-2, "moe_create: %d tokens of %d experts, rows of %d and %d: more than 2^27 groups of 256", max_tokens, top_k,
                  n_embd, n_ff);
        return nullptr;
    }
    // (slots and row blocks of gate and up; at fewer pairs, where tiles hold 32, slots are at most 3 / 2 n_experts)
    if (((long long)(pairs / 64) + n_experts) * ((n_ff + 63) / 64) > kMoeBlocks) {
        lib_error(-2, "moe_create: %d tokens of %d of %d experts, rows of %d: too many workgroups for a launch", max_tokens,
                  top_k, n_experts, n_ff);
        return nullptr;
    }
    if (!lib_ready("moe_create") || !moe_prepare<MoeQ6K>() || !moe_prepare<MoeQ80>() || !moe_prepare<MoeQ50>()) return nullptr;
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
    const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t sizes[7] = {4 * pairs, 4 * pairs, 4 * pairs, sizeof(MoeTile) * moe_slots(pairs, n_experts, 32),
                             kMoeRec * (records + 8), 4 * pairs * n_embd, sizeof(int32_t)};
    size_t total = 0, at[7];
    for (int i = 0; i < 7; ++i) {
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
    p->routed = (int32_t *)(p->mem + at[6]);
    if (!lib_hip(hipMemcpy(p->routed, &p->m, sizeof(p->m), hipMemcpyHostToDevice), "moe_create")) {
        (void)hipFree(p->mem);
        delete p;
        return nullptr;
    }
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
    // (a sort, where one follows, writes the tokens)
    const int now = moe_sorted(p, m) != 0 ? -1 : m;
    if (m == 0) {
        if (!lib_hip(launch_moe_assign(nullptr, nullptr, nullptr, nullptr, 0, p->n_experts, p->routed, 0,
                                       (hipStream_t)stream), "moe_route"))
            return 0;
    } else {
        RouteArgs a = {};
        a.scores = scores;
        a.bias = bias;
        a.ids = p->ids;
        a.ids_out = ids;
        a.routed = p->routed;
        a.now = now;
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
    if (!lib_hip(launch_moe_assign(ids, weights, p->ids, p->weights, m * p->top_k, p->n_experts, p->routed,
                                   moe_sorted(p, m) != 0 ? -1 : m, (hipStream_t)stream), "moe_assign"))
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
