// Attention of a step's tokens over the paged cache, by the plan of
// attn_plan.h: out = sum_j p_j V_j / sum_j p_j, p_j = exp(scale q.K_j - m), one
// pass over the keys with a running reference m and sum.
//
// Both products run on the matrix cores with the keys as the rows of the
// first operand, so that a query row is one column, held by the four lanes
// l, l + 16, l + 32, l + 48 through everything:
//   S^T = K Q^T   (16 keys x 16 query rows a tile): lane l gets, for query row
//                 l % 16, the keys 4 (l / 16) + r, r = 0..3;
//   O^T = V^T P^T (16 values x 16 query rows): the weights a lane has are the
//                 weights it must supply, in an order of keys that the V
//                 operand follows; no exchange between lanes.
// K and V come into LDS by DMA (16-byte pieces of a row permuted so that the
// reads below spread over the banks); V is read transposed (ds_read_..._tr).
//
// Arithmetic.  F16 and Q8_0: q (after an exact power-of-two scaling of its row
// that keeps both parts in range) and the weights as two f16 parts, high and
// rest, 22 bits together, against f16 values or the integer codes (exact in
// f16); two products each, f32 sums, at twice the matrix work, which stays under
// the time of the loads wherever few rows share them.  A single f16 part would
// lose 2^-11 of every weight.  Q8_0 scales are applied to the partial sums of a
// block (K) and to the weights (V).  F32: the f32 matrix instructions.
//
// A part's finest step is 2^-24, so a weight below 2^-2 has fewer than 22 bits;
// how many it has is a matter of the reference m in 2^(s - m + 10).  One that only
// ever rises to the row's maximum leaves the keys behind a strong one (an
// attention sink, whose value may well be next to zero) with few bits or none.  So
// m follows the scores of the tile at hand: it moves to the tile's maximum, and
// the row's sums are rescaled, where that is 2^5 above m or 2^13 below.  With t
// the largest of a row's weights in a tile of 32 keys, a weight w there is off by
// at most 2^-22 w, or 2^-22 t where that is more, and where t is the largest of
// the row so far by 2^-34 t.  (Raised at 2^4 instead of 2^6 chunks take 1 to 2 %
// longer; lowered at 2^10 instead of 2^14 2 to 9 %, as tiles that no row has to
// move for are looked at.)
//
// Q8_0 values.  Few rows: the parts are of weight times scale, with a reference
// for each row and block that follows in the same way, so a large scale costs
// nothing but its own block, and only rows that give its key weight.  Many rows
// share the values: those are code times scale in two f16 parts, the rest times
// 2^11, which hold any f16 scale's values whole at 2^15 for the largest so far.
// (Unscaled rests lost 2^-12 of a value 2^28 below it.  Single tokens as fast as
// with one unit for a wave's scales; 17 to 32 rows and chunks 2 to 4 % slower.)
//
// What bounds it, at head size 128 and 8 kv heads, measured:
//   few rows (single tokens, no sharing): the loads.  f16 5.5 TB/s, Q8_0 4.9,
//     f32 6.0 (a large copy: 5.1); 24 sequences of 200 to 12000 f16 keys 110 us;
//   many rows (a shared run, a chunk of tokens): matrix and vector instructions
//     together.  4 x 512 tokens behind 8192 f16 keys 490 us: 1.2 PFLOP/s of
//     matrix instructions (two for each product; a loop of nothing but them on
//     random operands reaches 1.75 on this card, a large library product 1.1);
//     MFMA 55 % of the cycles, waves wait 23 % and contend for issue 36 %;
//   short calls: a chain of loads (item -> page -> keys, item -> token -> query),
//     the first tile and the join of the waves, 5 to 7 us.
#include <hip/hip_runtime.h>

#include "gemm_common.h"
#include "kv.h"
#include "lib.h"

namespace exq {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
// The window around a row's reference: base-2 exponents above and below it.
constexpr float kUp = 5.0f, kDown = 13.0f;
// What the rest of a Q8_0 value beside its high part is kept times (many rows).
constexpr float kRest = 2048.0f;

struct AttnArgs {
    const float *q;
    float *out;
    const int32_t *head;
    float *part;
    KvView kv;
    float scale;
    int group;
    size_t part_cap;
    long long work, joins;  // items and joined rows, times kv heads; -1 (a captured call): as the plan says
};

// Sizes of a tile of TT keys: a unit is its K or its V rows in LDS.
template <int TYPE, int DIM>
struct Geo {
    static constexpr int TT = TYPE == kTypeF32 ? 16 : 32;
    static constexpr int HALVES = TT / 16;
    static constexpr int RB = TYPE == kTypeF32 ? DIM * 4 : TYPE == kTypeF16 ? DIM * 2 : DIM;  // row bytes
    static constexpr int CPR = RB / 16;                                                      // 16-byte pieces
    static constexpr int NB = DIM / 32;
    static constexpr int SB = TYPE == kTypeQ8_0 ? 2 * NB : 0;  // scale bytes of a row
    static constexpr int UNIT = TT * (RB + SB);
    static constexpr int CODE_OPS = (16 * RB + 1023) / 1024;  // DMA instructions for 16 rows
    static constexpr int HALF_OPS = CODE_OPS + (SB ? 1 : 0);
    static constexpr int OPS = HALVES * HALF_OPS;
    static constexpr int ND = DIM / 16;
    // few rows: each wave has its own ring of units; many rows: tiles shared by the workgroup
    static constexpr int RING = UNIT * 16 <= 80 * 1024 ? 4 : 2;
    static constexpr int SHARED = 4;
    static constexpr int TILE16 = 32 * DIM * 2;  // a unit's values as f16
    static constexpr int RT = DIM == 256 ? 1 : 2;  // 16-row tiles of a wave, many rows at most
    // Many rows with one tile a wave: not for Q8_0 but at 128, where two workgroups of 32 (64, 96: 53 and 81 ns a key
    // against 59 and 88) or four of 16 (256: 259 and 262) are faster.
    static constexpr bool ONE = TYPE != kTypeQ8_0 || DIM == 128;
    static constexpr int MANY = ONE || RT > 1 ? SHARED * 2 * UNIT + (SB ? 3 * TILE16 : 0) : 0;  // (Q8_0: codes of K, both parts of V)
    // 17 to 32 rows as few: with f16 no faster than the shared tiles (128: 56 and 57 ns a key), else near twice
    // (Q8_0 47 and 86, f32 101 and 169).
    static constexpr bool PAIR = RT == 2 && TYPE != kTypeF16;
    static constexpr int LDS = 4 * RING * UNIT > MANY ? 4 * RING * UNIT : MANY;
    static constexpr int MERGE = 4 * 16 * (DIM + 2) * 4;
    static constexpr int ODD = LDS > MERGE ? LDS : MERGE;  // marks of values that are not finite, a wave each
    static constexpr int ODD_WORDS = TT * NB;
    static constexpr int LDS_BYTES = ODD + 4 * ODD_WORDS * 4;
    static constexpr int PER_CU = LDS_BYTES <= 80 * 1024 ? 2 : 1;  // workgroups that LDS leaves room for
    // Registers for three where there is room for them (40 Q8_0 sequences behind 5000 tokens: 33 us with two, 28).
    static constexpr int WAVES = DIM == 64 ? 3 : PER_CU;
};

// Piece permutation of row `row` of a tile: piece c lies at c ^ swz.  Chosen so
// that 16 rows read at one piece (K), or 8 rows at two neighbouring pieces and
// 16 rows at one (V, transposed reads of 16 and 8 bits), or 4 rows 4 apart at
// 4 pieces (V, F32), fall on different banks of 64 (a quarter of the LDS cycles
// are conflicts all the same; LDS is busy a fifth of the time).
template <int TYPE, int DIM, bool V>
__device__ __forceinline__ int swz(int row) {
    if (TYPE == kTypeF32) {
        if (DIM == 96) return (row >> 1) & 7;
        return ((row >> 2) & 3) << 2 | (row & 3);
    }
    if (TYPE == kTypeF16) {
        if (DIM == 64) return ((row >> 1) & 3) << 1 | ((row >> 3) & 1);
        if (DIM == 96) return ((row >> 2) & 1) << 1 | ((row >> 3) & 1);
        return (row & 7) << 1 | ((row >> 3) & 1);
    }
    if (V) {
        const int b4 = (row >> 4) & 1;
        if (DIM == 64) return ((row >> 2) & 1) | b4 << 1;
        if (DIM == 96) return b4;
        if (DIM == 128) return ((row >> 1) & 3) | b4 << 2;
        return (row & 7) | b4 << 3;
    }
    if (DIM == 64) return (row >> 2) & 3;
    if (DIM == 96) return (row >> 3) & 1;
    if (DIM == 128) return (row >> 1) & 7;
    return row & 15;
}

__device__ __forceinline__ float xor16(float v) {
    return __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(v), 0x401f));
}
// Maximum and sum over the four lanes of a query row.
__device__ __forceinline__ float col_max(float v) {
    v = fmaxf(v, xor16(v));
    return fmaxf(v, shfl_xor_f(v, 32));
}
__device__ __forceinline__ float col_sum(float v) {
    v += xor16(v);
    return v + shfl_xor_f(v, 32);
}

__device__ __forceinline__ float wave_max(float v) {
    return col_max(row16_max(v));
}

__device__ __forceinline__ float wave_sum_f32(float v) {
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) v += reduce_partner(v, off);
    return col_sum(v);
}

// High part and rest of eight values.  The factor is one the compiler does not
// know, so that x - hi is one v_fma_mix_f32 and not a conversion and a
// subtraction.
__device__ __forceinline__ void split8(const float (&x)[8], v8h &hi, v8h &lo) {
    typedef float v2f __attribute__((ext_vector_type(2)));
    float minus = -1.0f;
    asm("" : "+v"(minus));
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const h2 h = __builtin_convertvector((v2f{x[j], x[j + 1]}), h2);
        const h2 l = __builtin_convertvector((v2f{fmaf((float)h[0], minus, x[j]), fmaf((float)h[1], minus, x[j + 1])}), h2);
        hi[j] = h[0];
        hi[j + 1] = h[1];
        lo[j] = l[0];
        lo[j + 1] = l[1];
    }
}

// The same of eight small integers times f, the rest times kRest.
__device__ __forceinline__ void split8(const v8h &q, float f, v8h &hi, v8h &lo) {
    typedef float v2f __attribute__((ext_vector_type(2)));
    float minus = -kRest;
    asm("" : "+v"(minus));
    const auto times = [&q](int j, float by) { return fmaf((float)q[j], by, 0.0f); };  // (one v_fma_mix_f32)
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const h2 h = __builtin_convertvector((v2f{times(j, f), times(j + 1, f)}), h2);
        const h2 l = __builtin_convertvector(
            (v2f{fmaf((float)h[0], minus, times(j, f * kRest)), fmaf((float)h[1], minus, times(j + 1, f * kRest))}), h2);
        hi[j] = h[0];
        hi[j + 1] = h[1];
        lo[j] = l[0];
        lo[j + 1] = l[1];
    }
}

// Four signed bytes as f16 (exact): 1024 + (byte + 128) built by v_perm, minus 1152.
__device__ __forceinline__ void bytes_h4(uint32_t w, _Float16 *o) {
    const uint32_t u = w ^ 0x80808080u;
    h2 p[2];
    bytes_to_h2(u, 0x64646464u, p);
    const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    p[0] = p[0] - off;
    p[1] = p[1] - off;
    o[0] = p[0][0];
    o[1] = p[0][1];
    o[2] = p[1][0];
    o[3] = p[1][1];
}
__device__ __forceinline__ v8h bytes_h8(uint32_t a, uint32_t b) {
    _Float16 o[8];
    bytes_h4(a, o);
    bytes_h4(b, o + 4);
    return v8h{o[0], o[1], o[2], o[3], o[4], o[5], o[6], o[7]};
}

__device__ __forceinline__ v4f mfma16(v8h a, v8h b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v4f mfma4(float a, float b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

typedef __attribute__((address_space(3))) v4s lds_v4s;
typedef __attribute__((address_space(3))) v2i lds_v2i;

// The lane number as a value the compiler knows nothing of: addresses made from
// it are not computed in front of the loops around, where they would hold
// registers all along.
__device__ __forceinline__ int here(int lane) {
    asm volatile("" : "+v"(lane));
    return lane;
}

// A barrier without the waits on memory of __syncthreads (the DMAs of later tiles stay in flight).
__device__ __forceinline__ void workgroup_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ void lds_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The token of row r of an item, and where its output goes.
__device__ __forceinline__ const PlanToken *token_of(const AttnArgs &a, const AttnItem &it, int r) {
    return reinterpret_cast<const PlanToken *>(a.head) - ((it.row0 + r) / a.group + 1);
}
__device__ __forceinline__ size_t row_at(const AttnArgs &a, const AttnItem &it, int h, int r, int dim) {
    return (((size_t)token_of(a, it, r)->order * a.kv.n_kv + h) * a.group + (it.row0 + r) % a.group) * dim;
}

// Where a piece of work reads: the pages of one kv head of one layer.
struct Source {
    const __attribute__((address_space(4))) int32_t *pages;  // page of position p: pages[p >> shift]
    const uint8_t *base;                                      // the layer's, at this head's K
    size_t page_bytes;
    uint32_t head_bytes, v_off;
    int shift, last;  // last: the highest page index there is
};

template <int TYPE, int DIM>
struct Loader {
    using G = Geo<TYPE, DIM>;
    // The page of position p.  Asked for one tile ahead of its use.
    static __device__ __forceinline__ int page(const Source &s, int p) { return s.pages[min(p >> s.shift, s.last)]; }
    // 16 rows of K (which = 0) or V at position p, half hf of the unit at LDS byte `to`: their sub-operations sub0 to
    // sub0 + N - 1 of HALF_OPS, a DMA instruction each (with Q8_0 the last one is the scales).
    template <int N>
    static __device__ __forceinline__ void rows(const Source &s, int page, int which, int hf, int sub0, int p, uint32_t to, int lane) {
        const v4u rs = rsrc_words(s.base + (size_t)(uint32_t)page * s.page_bytes + (which ? s.v_off : 0u), s.head_bytes);
        const uint32_t off = (uint32_t)(p & ((1 << s.shift) - 1));
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (G::SB != 0 && k == G::CODE_OPS) {
                const uint32_t so = ((uint32_t)DIM << s.shift) + off * G::SB;
                if (lane < G::SB) dma16(to + G::TT * G::RB + hf * 16 * G::SB, lane * 16, rs, so);
                continue;
            }
            const int at = (sub0 + k) * 1024 + lane * 16, row = at / G::RB, piece = at % G::RB / 16;
            const int sw = which ? swz<TYPE, DIM, true>(hf * 16 + row) : swz<TYPE, DIM, false>(hf * 16 + row);
            const uint32_t vo = (uint32_t)(row * G::RB + ((piece ^ sw) * 16)), dst = to + hf * 16 * G::RB + (sub0 + k) * 1024;
            if (16 * G::RB % 1024 == 0 || k < G::CODE_OPS - 1) dma16(dst, vo, rs, off * G::RB);
            else if (lane < 16 * G::RB % 1024 / 16) dma16(dst, vo, rs, off * G::RB);
        }
    }
    // A whole unit by one wave.
    struct Pages {
        int at[G::HALVES];
    };
    static __device__ __forceinline__ Pages pages(const Source &s, int p0) {
        Pages pg;
#pragma unroll
        for (int hf = 0; hf < G::HALVES; ++hf) pg.at[hf] = page(s, p0 + 16 * hf);
        return pg;
    }
    static __device__ __forceinline__ void unit(const Source &s, const Pages &pg, int which, int p0, uint32_t to, int lane) {
#pragma unroll
        for (int hf = 0; hf < G::HALVES; ++hf) rows<G::HALF_OPS>(s, pg.at[hf], which, hf, 0, p0 + 16 * hf, to, lane);
    }
    // A wave's part of a tile's two units: 16 rows of one of them, or half of those (every wave the same number).
    static constexpr int SHARE = G::HALVES == 2 ? G::HALF_OPS : G::CODE_OPS / 2;
    static_assert(G::HALVES == 2 || (G::SB == 0 && G::CODE_OPS % 2 == 0), "equal shares");
    static __device__ __forceinline__ int share_at(int p0, int wave) { return G::HALVES == 2 ? p0 + 16 * (wave & 1) : p0; }
    static __device__ __forceinline__ void share(const Source &s, int page, int p0, uint32_t to, int wave, int lane) {
        rows<SHARE>(s, page, wave >> 1, G::HALVES == 2 ? wave & 1 : 0, G::HALVES == 2 ? 0 : (wave & 1) * SHARE, share_at(p0, wave),
                    to + (wave >> 1) * G::UNIT, lane);
    }
};

// A wave's query rows: RT tiles of 16, row l % 16 of a tile on lane l.
template <int TYPE, int DIM, int RT, bool MANY>
struct Rows {
    using G = Geo<TYPE, DIM>;
    static constexpr bool BLOCKS = TYPE == kTypeQ8_0 && !MANY;         // the parts are of weight times scale, a block each
    static constexpr bool FOLLOW = TYPE != kTypeF32 && !BLOCKS;        // the parts are of the weights
    v8h qh[TYPE == kTypeF32 ? 1 : RT][TYPE == kTypeF32 ? 1 : G::NB], ql[TYPE == kTypeF32 ? 1 : RT][TYPE == kTypeF32 ? 1 : G::NB];
    v4f qf[TYPE == kTypeF32 ? RT : 1][TYPE == kTypeF32 ? G::ND : 1];
    float top[RT], rs[RT], m[RT], l[RT];  // score factor (positive); reference (a base-2 exponent), this lane's part of the sum
    int lim[RT];                 // positions below are seen
    v4f acc[RT][G::ND];
    static constexpr int kMostUp = 64;            // (the first tile with a value that is not zero finds it out of the window)
    float up[BLOCKS ? RT : 1][BLOCKS ? G::NB : 1];  // BLOCKS: acc of block b is times this power of two
    int ve;                                         // Q8_0, many rows: acc is in units of 2^(ve - 8)
    float s[RT][G::HALVES][4], p[RT][G::HALVES][4];  // a tile's scores, its weights

    __device__ __forceinline__ void load(const AttnArgs &a, const AttnItem &it, int h, int row_from, int lane) {
        const int g = lane >> 4;
        // a negative scale turns q around; zero makes q zero
        const float sign = a.scale < 0.0f ? -1.0f : a.scale == 0.0f ? 0.0f : 1.0f;
        const float scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * kLog2e;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int r = min(row_from + 16 * t + (lane & 15), it.n_rows - 1);
            lim[t] = it.causal ? min(it.key1, token_of(a, it, r)->order_pos + 1) : it.key1;
            const float *q = a.q + row_at(a, it, h, r, DIM);
            if constexpr (TYPE == kTypeF32) {
#pragma unroll
                for (int c = 0; c < G::ND; ++c) qf[t][c] = sign * *reinterpret_cast<const v4f *>(q + c * 16 + g * 4);
                rs[t] = fmaxf(scale, 1.17549435e-38f);
            } else {
                float x[G::NB][8], top = 0.0f;
#pragma unroll
                for (int c = 0; c < G::NB; ++c) {
                    const v4f u = *reinterpret_cast<const v4f *>(q + c * 32 + g * 8);
                    const v4f v = *reinterpret_cast<const v4f *>(q + c * 32 + g * 8 + 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        x[c][j] = sign * u[j];
                        x[c][4 + j] = sign * v[j];
                        top = fmaxf(top, fmaxf(fabsf(u[j]), fabsf(v[j])));
                    }
                }
                top = col_max(top);
                // the row's largest value in [2^14, 2^15)
                const int e = top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) - 15 : 0;
#pragma unroll
                for (int c = 0; c < G::NB; ++c) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[c][j] = ldexpf(x[c][j], -e);
                    split8(x[c], qh[t][c], ql[t][c]);
                }
                // (not zero: a masked score is -infinity times this)
                rs[t] = fmaxf(ldexpf(scale, e), 1.17549435e-38f);
            }
            m[t] = -INFINITY;
            l[t] = 0.0f;
#pragma unroll
            for (int d = 0; d < G::ND; ++d) acc[t][d] = v4f{0, 0, 0, 0};
            if constexpr (BLOCKS) {
#pragma unroll
                for (int b = 0; b < G::NB; ++b) up[t][b] = ldexpf(1.0f, kMostUp);
            }
        }
        ve = -24;
    }

    // Scores of the K unit at ku; k16: its codes as f16 (Q8_0, many rows).
    __device__ __forceinline__ void scores(const uint8_t *ku, const uint8_t *k16, int lane) {
        const int g = lane >> 4, c16 = lane & 15;
#pragma unroll
        for (int hf = 0; hf < G::HALVES; ++hf) {
            const int row = hf * 16 + c16, sw = swz<TYPE, DIM, false>(row);
            const uint8_t *kr = ku + row * G::RB;
            v4f o[RT];
#pragma unroll
            for (int t = 0; t < RT; ++t) o[t] = v4f{0, 0, 0, 0};
            if constexpr (TYPE == kTypeF32) {
#pragma unroll
                for (int c = 0; c < G::ND; ++c) {
                    const v4f k = *reinterpret_cast<const v4f *>(kr + (((c * 4 + g) ^ sw) * 16));
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int t = 0; t < RT; ++t) o[t] = mfma4(k[j], qf[t][c][j], o[t]);
                }
            } else if constexpr (TYPE == kTypeF16) {
#pragma unroll
                for (int c = 0; c < G::NB; ++c) {
                    const v8h k = *reinterpret_cast<const v8h *>(kr + (((c * 4 + g) ^ sw) * 16));
#pragma unroll
                    for (int t = 0; t < RT; ++t) o[t] = mfma16(k, ql[t][c], o[t]);
#pragma unroll
                    for (int t = 0; t < RT; ++t) o[t] = mfma16(k, qh[t][c], o[t]);
                }
            } else {
                const _Float16 *ds = reinterpret_cast<const _Float16 *>(ku + G::TT * G::RB) + (hf * 16 + g * 4) * G::NB;
#pragma unroll
                for (int c = 0; c < G::NB; ++c) {
                    v8h k;
                    if (k16 != nullptr) {
                        k = *reinterpret_cast<const v8h *>(k16 + row * DIM * 2 + (((c * 4 + g) ^ swz<kTypeF16, DIM, false>(row)) * 16));
                    } else {
                        const v2u w = *reinterpret_cast<const v2u *>(kr + (((c * 2 + (g >> 1)) ^ sw) * 16) + (g & 1) * 8);
                        k = bytes_h8(w[0], w[1]);
                    }
#pragma unroll
                    for (int t = 0; t < RT; ++t) {
                        v4f b = mfma16(k, ql[t][c], v4f{0, 0, 0, 0});
                        b = mfma16(k, qh[t][c], b);
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[t][r] = fmaf((float)ds[r * G::NB + c], b[r], o[t][r]);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[t][hf][r] = o[t][r];
        }
    }

    // Positions at or past a row's limit get no weight.
    __device__ __forceinline__ void mask(int p0, int lane) {
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int hf = 0; hf < G::HALVES; ++hf)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (p0 + hf * 16 + (lane >> 4) * 4 + r >= lim[t]) s[t][hf][r] = -INFINITY;
    }

    __device__ __forceinline__ void rescale(float c, int t) {
#pragma unroll
        for (int d = 0; d < G::ND; ++d) acc[t][d] *= c;
    }

    // This lane's largest scores.
    __device__ __forceinline__ void tops() {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            top[t] = -INFINITY;
#pragma unroll
            for (int hf = 0; hf < G::HALVES; ++hf)
#pragma unroll
                for (int r = 0; r < 4; ++r) top[t] = fmaxf(top[t], s[t][hf][r]);
            top[t] *= rs[t];
        }
    }

    // A row's reference moves to the largest score of its tile where that is out of the window: by the row's own keys, no
    // other row has a say.  It is lowered as long as the weights' sum stays below 2^96 (values: 2^16 at most).  It is a
    // whole number, so that the sums keep all their bits however often it moves.
    __device__ __forceinline__ void follow() {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const float gap = top[t] - m[t];
            const bool out = !FOLLOW ? gap > kUp : fabsf(gap + (kDown - kUp) / 2) > (kDown + kUp) / 2;
            if (__builtin_amdgcn_ballot_w64(out) != 0) {
                const float row = col_max(top[t]);
                const bool lower = FOLLOW && row < m[t] - kDown && row > -INFINITY &&
                                   col_max(l[t]) * __builtin_amdgcn_exp2f(m[t] - row) < 0x1p96f;
                const float mn = row > m[t] + kUp || lower ? rintf(row) : m[t];
                // (-infinity, the first: zero)
                const float c = m[t] == mn ? 1.0f : ldexpf(1.0f, (int)fmaxf(-200.0f, fminf(200.0f, m[t] - mn)));
                m[t] = mn;
                l[t] *= c;
                rescale(c, t);
            }
        }
    }

    // Scores become weights.
    __device__ __forceinline__ void weights() {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const float off = m[t] == -INFINITY ? 0.0f : m[t] - (TYPE == kTypeF32 ? 0.0f : 15.0f - kUp);
#pragma unroll
            for (int hf = 0; hf < G::HALVES; ++hf)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    p[t][hf][r] = __builtin_amdgcn_exp2f(fmaf(s[t][hf][r], rs[t], -off));
                    l[t] += p[t][hf][r];
                }
        }
    }

    // acc += V^T P^T for f16 values in rows of DIM, or (PARTS) for their high parts at vu and the rests, times kRest, at
    // vl: those meet the weights / kRest, which loses no more of a weight than its own rest has lost.  The product of
    // the two rests (2^-22 of a value) is left out.
    template <bool PARTS>
    __device__ __forceinline__ void values16(const uint8_t *vu, const uint8_t *vl, int lane) {
        const int g = lane >> 4, c16 = lane & 15;
        v8h ph[RT], pl[RT], ps[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const float x[8] = {p[t][0][0], p[t][0][1], p[t][0][2], p[t][0][3], p[t][1][0], p[t][1][1], p[t][1][2], p[t][1][3]};
            split8(x, ph[t], pl[t]);
            if (PARTS) ps[t] = ph[t] * (_Float16)(1.0f / kRest);
        }
        const int row = g * 4 + (c16 >> 2), sw = swz<kTypeF16, DIM, true>(row);  // the same for row + 16
        const auto read = [&](const uint8_t *from, int d) {
            const uint8_t *at = from + row * DIM * 2 + (((d * 2 + ((c16 >> 1) & 1)) ^ sw) * 16) + (c16 & 1) * 8;
            const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)at);
            const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(at + 16 * DIM * 2));
            return __builtin_bit_cast(v8h, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        };
#pragma unroll
        for (int d = 0; d < G::ND; ++d) {
            const v8h v = read(vu, d);
            if (PARTS) {
                const v8h rest = read(vl, d);
#pragma unroll
                for (int t = 0; t < RT; ++t) acc[t][d] = mfma16(rest, ps[t], acc[t][d]);
            }
#pragma unroll
            for (int t = 0; t < RT; ++t) acc[t][d] = mfma16(v, pl[t], acc[t][d]);
#pragma unroll
            for (int t = 0; t < RT; ++t) acc[t][d] = mfma16(v, ph[t], acc[t][d]);
        }
    }

    // This lane's largest finite scale of the V unit at vu (the lanes together: the unit's).
    static __device__ __forceinline__ float finite_top(const uint8_t *vu, int lane) {
        const _Float16 *d = reinterpret_cast<const _Float16 *>(vu + G::TT * G::RB);
        float top = 0.0f;
        for (int k = lane; k < G::TT * G::NB; k += 64) {
            const float x = fabsf((float)d[k]);
            if (x < INFINITY) top = fmaxf(top, x);
        }
        return top;
    }

    // Q8_0, many rows: the unit of acc is raised to 2^(e - 8) where the largest scale `top` (of the wave's lanes together)
    // exceeds 2^e, so that a value in it is below 2^15; its two parts (down to 2^-35) then hold it whole, whatever the
    // other scales are.  A scale that is not finite makes its block's sums NaN in any unit, and has no say in the others'.
    __device__ __forceinline__ void raise_unit(float top, const uint8_t *vu, int lane) {
        if (__builtin_amdgcn_ballot_w64(top > ldexpf(1.0f, ve)) == 0) return;
        if (__builtin_amdgcn_ballot_w64(top == INFINITY) != 0) top = finite_top(vu, lane);
        const int e = __builtin_amdgcn_readfirstlane(__builtin_amdgcn_frexp_expf(wave_max(top)));
        if (e <= ve) return;
#pragma unroll
        for (int t = 0; t < RT; ++t) rescale(ldexpf(1.0f, ve - e), t);
        ve = e;
    }

    // acc += V^T P^T for the V unit at vu.
    __device__ __forceinline__ void values(const uint8_t *vu, int lane) {
        const int g = lane >> 4, c16 = lane & 15;
        if constexpr (TYPE == kTypeF32) {
#pragma unroll
            for (int d = 0; d < G::ND; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = g * 4 + r, sw = swz<TYPE, DIM, true>(row);
                    const float v = *reinterpret_cast<const float *>(vu + row * G::RB + (((d * 4 + (c16 >> 2)) ^ sw) * 16) + (c16 & 3) * 4);
#pragma unroll
                    for (int t = 0; t < RT; ++t) acc[t][d] = mfma4(v, p[t][0][r], acc[t][d]);
                }
        } else if constexpr (TYPE == kTypeF16) {
            values16<false>(vu, nullptr, lane);
        } else {
            // this lane's keys: 4 g + r of both halves; their blocks' scales, two to a word
            const uint32_t *ds = reinterpret_cast<const uint32_t *>(vu + G::TT * G::RB) + g * 2 * G::NB;
            uint32_t sc[2][2 * G::NB];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                for (int i = 0; i < 2 * G::NB; ++i) sc[hf][i] = ds[hf * 8 * G::NB + i];
            const int o = c16 >> 1, row = (o < 4 ? g * 4 + o : 16 + g * 4 + o - 4), sw = swz<TYPE, DIM, true>(row);
            // Several blocks a branch: one for each would keep their products apart (5 to 13 % of the time), and all are
            // too many registers with two tiles of rows or eight blocks.
            constexpr int GROUP = G::NB == 2 ? 2 / RT : RT == 1 && G::NB <= 4 ? G::NB : 2;
#pragma unroll
            for (int b0 = 0; b0 < G::NB; b0 += GROUP) {
                float x[GROUP][RT][8], big[GROUP][RT];
                bool out = false;
#pragma unroll
                for (int k = 0; k < GROUP && b0 + k < G::NB; ++k)
#pragma unroll
                    for (int t = 0; t < RT; ++t) {
                        big[k][t] = 0.0f;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int i = j % 4 * G::NB + b0 + k;
                            const float d = fmaf((float)__builtin_bit_cast(h2, sc[j / 4][i / 2])[i % 2], up[t][b0 + k], 0.0f);
                            x[k][t][j] = p[t][j / 4][j % 4] * d;
                            big[k][t] = fmaxf(big[k][t], fabsf(x[k][t][j]));
                        }
                        out |= !in_window(big[k][t]);
                    }
                if (__builtin_amdgcn_ballot_w64(out) != 0) {
#pragma unroll
                    for (int k = 0; k < GROUP && b0 + k < G::NB; ++k)
#pragma unroll
                        for (int t = 0; t < RT; ++t) fit(t, b0 + k, col_max(big[k][t]), x[k][t]);
                }
#pragma unroll
                for (int k = 0; k < GROUP && b0 + k < G::NB; ++k) {
                    v8h ph[RT], pl[RT];
#pragma unroll
                    for (int t = 0; t < RT; ++t) split8(x[k][t], ph[t], pl[t]);
#pragma unroll
                    for (int d = 2 * (b0 + k); d < 2 * (b0 + k) + 2; ++d) {
                        const uint8_t *at = vu + row * G::RB + ((d ^ sw) * 16) + (c16 & 1) * 8;
                        const v2i w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i *)at);
                        const v8h v = bytes_h8((uint32_t)w[0], (uint32_t)w[1]);
#pragma unroll
                        for (int t = 0; t < RT; ++t) acc[t][d] = mfma16(v, pl[t], acc[t][d]);
#pragma unroll
                        for (int t = 0; t < RT; ++t) acc[t][d] = mfma16(v, ph[t], acc[t][d]);
                    }
                }
            }
        }
    }

    // BLOCKS: whether a tile's largest weight times scale leaves its parts their bits, and the factor of block b that
    // puts it, `big`, between 2^9 and 2^10 where not.  A row's own, from its own keys (one that is not finite makes the
    // block NaN whatever the factor; zeros need none; sums stay below 2^102 n).
    static __device__ __forceinline__ bool in_window(float v) { return v <= 32768.0f && v >= 0.125f; }
    __device__ __forceinline__ void fit(int t, int b, float big, float (&x)[8]) {
        if (in_window(big) || big == 0.0f || !(big < INFINITY)) return;
        const int had = __builtin_amdgcn_frexp_expf(up[t][b]) - 1;
        const int more = min(10 - __builtin_amdgcn_frexp_expf(big), kMostUp - had);
        const float c = ldexpf(1.0f, more);
#pragma unroll
        for (int d = 2 * b; d < 2 * b + 2; ++d) acc[t][d] *= c;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= c;
        up[t][b] *= c;
    }

    // The sums that a key's values marked in `odd` (NB words a key) belong to become NaN for the rows that see it.
    __device__ __forceinline__ void spoil(const uint32_t *odd, int p0, int lane) {
        const int g = lane >> 4;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            uint32_t w[G::NB] = {};
#pragma unroll 1
            for (int k = 0; k < G::TT && p0 + k < lim[t]; ++k)
#pragma unroll
                for (int b = 0; b < G::NB; ++b) w[b] |= odd[k * G::NB + b];
#pragma unroll
            for (int d = 0; d < G::ND; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (w[d / 2] >> ((d & 1) * 16 + g * 4 + j) & 1) acc[t][d][j] = __builtin_nanf("");
        }
    }

    // No row of the wave sees this position or any behind it.
    __device__ __forceinline__ int last_limit() const {
        int v = lim[RT - 1];
#pragma unroll
        for (int t = 0; t < RT; ++t) v = max(v, lim[t]);
        return __builtin_amdgcn_readlane(v, 15);
    }

    // acc in units of one, l the row's whole sum.  What is not finite becomes NaN: an infinite value gives infinity or NaN
    // by the signs of the weights' rests, and NaN in a tile at the causal limit.
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            l[t] = col_sum(l[t]);
            if constexpr (BLOCKS) {
#pragma unroll
                for (int d = 0; d < G::ND; ++d) acc[t][d] *= 1.0f / up[t][d / 2];
            } else if (TYPE == kTypeQ8_0) {
                rescale(ldexpf(1.0f, ve - 8), t);
            }
#pragma unroll
            for (int d = 0; d < G::ND; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[t][d][j] = fmaf(acc[t][d][j], 0.0f, acc[t][d][j]);
        }
    }
};

// Slots past the last key may hold anything: their V rows (their scales) become zero in LDS.
template <int TYPE, int DIM>
__device__ __forceinline__ void clear_tail(uint8_t *vu, int valid, int tid, int n) {
    using G = Geo<TYPE, DIM>;
    if (TYPE == kTypeQ8_0) {
        for (int i = valid * G::SB / 2 + tid; i < G::TT * G::SB / 2; i += n)
            reinterpret_cast<uint16_t *>(vu + G::TT * G::RB)[i] = 0;
    } else {
        for (int i = valid * G::CPR + tid; i < G::TT * G::CPR; i += n) reinterpret_cast<v4u *>(vu)[i] = v4u{0, 0, 0, 0};
    }
}

// Whether the V unit at vu holds a value (a scale) that is not finite.
template <int TYPE, int DIM>
__device__ __forceinline__ bool odd_values(const uint8_t *vu, int lane) {
    using G = Geo<TYPE, DIM>;
    const uint8_t *at = TYPE == kTypeQ8_0 ? vu + G::TT * G::RB : vu;
    constexpr int n = TYPE == kTypeQ8_0 ? G::TT * G::SB : G::TT * G::RB;
    constexpr uint32_t lo = TYPE == kTypeF32 ? 0x7f800000u : 0x7c00u, hi = TYPE == kTypeF32 ? lo : lo << 16;
    bool bad = false;
#pragma unroll 2
    for (int i = lane * 4; i < n; i += 256) {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(at + i);
        bad |= (w & lo) == lo || (w & hi) == hi;
    }
    return __builtin_amdgcn_ballot_w64(bad) != 0;
}

// In a tile at the causal limit 0 * infinity must not reach the rows that do
// not see the key.  One wave marks the values that are not finite in `odd`
// (NB words a key, bit e % 32 of word e / 32 for value e; a Q8_0 scale marks its
// block) and makes them zero; spoil() then does to the rows that see them what
// the product would have done.
template <int TYPE, int DIM>
__device__ __forceinline__ void mark_odd(uint8_t *vu, uint32_t *odd, int lane) {
    using G = Geo<TYPE, DIM>;
    if (lane >= G::TT) return;
    const int sw = swz<TYPE, DIM, true>(lane);
#pragma unroll 1
    for (int b = 0; b < G::NB; ++b) {
        uint32_t w = 0;
        if (TYPE == kTypeQ8_0) {
            uint16_t *d = reinterpret_cast<uint16_t *>(vu + G::TT * G::RB) + lane * G::NB + b;
            if ((*d & 0x7c00u) == 0x7c00u) {
                w = ~0u;
                *d = 0;
            }
        } else {
            constexpr int es = TYPE == kTypeF32 ? 4 : 2;
#pragma unroll 1
            for (int j = 0; j < 32; ++j) {
                const int e = b * 32 + j;
                uint8_t *at = vu + lane * G::RB + (((e * es / 16) ^ sw) * 16) + e * es % 16;
                const bool bad = TYPE == kTypeF32 ? (*reinterpret_cast<uint32_t *>(at) & 0x7f800000u) == 0x7f800000u
                                                  : (*reinterpret_cast<uint16_t *>(at) & 0x7c00u) == 0x7c00u;
                if (!bad) continue;
                w |= 1u << j;
                if (TYPE == kTypeF32) *reinterpret_cast<uint32_t *>(at) = 0;
                else *reinterpret_cast<uint16_t *>(at) = 0;
            }
        }
        odd[lane * G::NB + b] = w;
    }
}

// Q8_0, many rows: a tile's K codes and V values become f16 in LDS once for all
// waves.  V: code * scale / unit (18 bits) as high part and rest times kRest.  Each wave
// multiplying its own operands out took twice the vector instructions.
template <int DIM>
__device__ __forceinline__ void expand(const uint8_t *ku, const uint8_t *vu, uint8_t *to, float unit, int tid) {
    using G = Geo<kTypeQ8_0, DIM>;
    constexpr int PIECES = 32 * DIM / 16;
#pragma unroll
    for (int k = 0; k < (PIECES + 255) / 256; ++k) {
        const int i = tid + 256 * k, row = i / G::CPR, c = i % G::CPR;
        if (PIECES % 256 != 0 && i >= PIECES) break;
        const int s16 = swz<kTypeF16, DIM, false>(row);
        uint8_t *o = to + row * DIM * 2;
        const int o0 = ((2 * c) ^ s16) * 16, o1 = ((2 * c + 1) ^ s16) * 16;
        const v4u kw = *reinterpret_cast<const v4u *>(ku + row * G::RB + ((c ^ swz<kTypeQ8_0, DIM, false>(row)) * 16));
        const v4u vw = *reinterpret_cast<const v4u *>(vu + row * G::RB + ((c ^ swz<kTypeQ8_0, DIM, true>(row)) * 16));
        *reinterpret_cast<v8h *>(o + o0) = bytes_h8(kw[0], kw[1]);
        *reinterpret_cast<v8h *>(o + o1) = bytes_h8(kw[2], kw[3]);
        const float f = (float)reinterpret_cast<const _Float16 *>(vu + G::TT * G::RB)[row * G::NB + c / 2] * unit;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const v8h q = bytes_h8(vw[2 * j], vw[2 * j + 1]);
            v8h hi, lo;
            split8(q, f, hi, lo);
            *reinterpret_cast<v8h *>(o + G::TILE16 + (j ? o1 : o0)) = hi;
            *reinterpret_cast<v8h *>(o + 2 * G::TILE16 + (j ? o1 : o0)) = lo;
        }
    }
}

// Few rows (at most 16 RT): the four waves take every fourth tile of keys each,
// on their own (no barrier), and join their sums at the end.
template <int TYPE, int DIM, int RT>
__device__ __forceinline__ void attend_few(const AttnArgs &a, const AttnItem &it, const Source &src, int h, uint8_t *lds,
                                           int wave, int lane) {
    using G = Geo<TYPE, DIM>;
    using L = Loader<TYPE, DIM>;
    Rows<TYPE, DIM, RT, false> w;
    const int tiles = (it.key1 - it.key0 + G::TT - 1) / G::TT;
    const int mine = (tiles - wave + 3) / 4, units = 2 * mine;
    const uint32_t ring = lds_addr(lds) + wave * G::RING * G::UNIT;
    uint8_t *ringp = lds + wave * G::RING * G::UNIT;
    const auto pos = [&](int u) { return it.key0 + (wave + 4 * (u >> 1)) * G::TT; };
    const auto issue = [&](int u, const typename L::Pages &pg) {
        if (u < units) L::unit(src, pg, u & 1, pos(u), ring + (u % G::RING) * G::UNIT, lane);
    };
    const auto arrive = [&](int u) {  // unit u is there; what was read before it may be overwritten
        if (u + G::RING - 2 < units) wait_dma<(G::RING - 2) * G::OPS>();
        else wait_dma<0>();
        lds_done();
    };
    static_assert(G::RING % 2 == 0, "the units asked for while tile i is computed are V of tile i + RING/2 - 1, K of the next");
    constexpr int ahead = G::RING / 2 - 1;
    typename L::Pages now = L::pages(src, pos(0)), then = now;
    for (int u = 0; u < G::RING - 1; ++u) {
        if (u > 0 && u % 2 == 0) now = L::pages(src, pos(u));
        issue(u, now);
    }
    then = L::pages(src, pos(2 * ahead + 2));
    w.load(a, it, h, 0, lane);  // (behind the first DMAs: one latency less; its loads wait for theirs)
    wait_dma<0>();
    // the first row's limit: a tile below it needs no mask
    const int first = it.causal ? __builtin_amdgcn_readfirstlane(w.lim[0]) : it.key1;
    for (int i = 0; i < mine; ++i) {
        const int p0 = pos(2 * i);
        const bool edge = p0 + G::TT > first;
        arrive(2 * i);
        issue(2 * (i + ahead) + 1, now);
        w.scores(ringp + (2 * i % G::RING) * G::UNIT, nullptr, lane);
        if (edge) w.mask(p0, lane);
        w.tops();
        w.follow();
        w.weights();
        arrive(2 * i + 1);
        issue(2 * (i + ahead) + 2, then);
        now = then;
        then = L::pages(src, pos(2 * (i + ahead) + 4));
        uint8_t *vu = ringp + ((2 * i + 1) % G::RING) * G::UNIT;
        if (edge) {
            if (p0 + G::TT > it.key1) {
                clear_tail<TYPE, DIM>(vu, it.key1 - p0, lane, 64);
                lds_done();
            }
            if (odd_values<TYPE, DIM>(vu, here(lane))) {
                uint32_t *odd = reinterpret_cast<uint32_t *>(lds + G::ODD) + wave * G::ODD_WORDS;
                mark_odd<TYPE, DIM>(vu, odd, here(lane));
                lds_done();
                w.spoil(odd, p0, here(lane));
            }
        }
        w.values(vu, lane);
    }
    w.finish();
    // join the waves, 16 rows at a time: [wave][row][DIM], then maxima and sums
    float *mo = reinterpret_cast<float *>(lds), *ml = mo + 4 * 16 * DIM;
    const int c = lane & 15, g = lane >> 4;
    const int tid = wave * 64 + lane;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        __syncthreads();
#pragma unroll
        for (int d = 0; d < G::ND; ++d) *reinterpret_cast<v4f *>(mo + (wave * 16 + c) * DIM + d * 16 + g * 4) = w.acc[t][d];
        if (g == 0) {
            ml[2 * (wave * 16 + c)] = w.m[t];
            ml[2 * (wave * 16 + c) + 1] = w.l[t];
        }
        __syncthreads();
        for (int i = tid; i < min(16, it.n_rows - 16 * t) * (DIM / 4); i += 256) {
            const int r = i / (DIM / 4), e = i % (DIM / 4) * 4;
            float m = -INFINITY, l = 0.0f;
#pragma unroll
            for (int v = 0; v < 4; ++v) m = fmaxf(m, ml[2 * (v * 16 + r)]);
            v4f o = {0, 0, 0, 0};
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const float mv = ml[2 * (v * 16 + r)];
                if (mv == -INFINITY && ml[2 * (v * 16 + r) + 1] == 0.0f) continue;  // no key of this wave's is seen
                const float f = __builtin_amdgcn_exp2f(mv - m);
                l += f * ml[2 * (v * 16 + r) + 1];
                o += f * *reinterpret_cast<const v4f *>(mo + (v * 16 + r) * DIM + e);
            }
            if (it.part < 0) {
                *reinterpret_cast<v4f *>(a.out + row_at(a, it, h, 16 * t + r, DIM) + e) = o / l;
            } else {
                const size_t ps = (size_t)(it.part + 16 * t + r) * a.kv.n_kv + h;
                *reinterpret_cast<v4f *>(a.part + ps * DIM + e) = o;
                if (e == 0) {
                    float *d = a.part + a.part_cap * DIM + 2 * ps;
                    d[0] = m;
                    d[1] = l;
                }
            }
        }
    }
    __syncthreads();
}

// Many rows: every wave has its own (RT tiles of 16), and all read the same
// tiles of keys.  The scores of tile i + 1 are computed in front of the values
// of tile i, so that matrix instructions and the exponentials of tile i can run
// side by side.
template <int TYPE, int DIM, int RT>
__device__ __forceinline__ void attend_many(const AttnArgs &a, const AttnItem &it, const Source &src, int h, uint8_t *lds,
                                            int wave, int lane) {
    using G = Geo<TYPE, DIM>;
    using L = Loader<TYPE, DIM>;
    Rows<TYPE, DIM, RT, true> w;
    const int mine = wave * 16 * RT;  // (past the last row: computed from that row, not stored)
    const int tiles = (it.key1 - it.key0 + G::TT - 1) / G::TT;
    const uint32_t base = lds_addr(lds);
    const auto unit_at = [&](int i) { return lds + (i % G::SHARED) * 2 * G::UNIT; };
    const auto page_of = [&](int i) { return L::page(src, L::share_at(it.key0 + i * G::TT, wave)); };
    const auto issue = [&](int i, int pg) {
        if (i < tiles) L::share(src, pg, it.key0 + i * G::TT, base + (i % G::SHARED) * 2 * G::UNIT, wave, lane);
    };
    for (int i = 0; i < G::SHARED - 1; ++i) issue(i, page_of(i));
    int next = page_of(G::SHARED - 1);
    w.load(a, it, h, mine, lane);  // (behind the first DMAs: one latency less; its loads wait for theirs)
    const int first = it.causal ? __builtin_amdgcn_readfirstlane(w.lim[0]) : it.key1;
    const int wave_last = it.causal ? w.last_limit() : it.key1;
    // (the workgroup's first row: the least limit of all waves)
    const int all_first = it.causal ? min(it.key1, token_of(a, it, 0)->order_pos + 1) : it.key1;
    wait_dma<0>();
    workgroup_barrier();
    uint8_t *wide = lds + G::SHARED * 2 * G::UNIT;  // Q8_0: f16 codes of the next tile's K, parts of this tile's V
    w.scores(unit_at(0), nullptr, lane);
    w.tops();
    for (int i = 0; i < tiles; ++i) {
        const int p0 = it.key0 + i * G::TT;
        uint8_t *vu = unit_at(i) + G::UNIT;
        if (i + G::SHARED - 2 < tiles) wait_dma<(G::SHARED - 3) * L::SHARE>();  // tile i + 1 is there
        else wait_dma<0>();
        lds_done();
        workgroup_barrier();
        issue(i + G::SHARED - 1, next);
        next = page_of(i + G::SHARED);
        if (p0 + G::TT > it.key1) {  // (the last tile, for all waves)
            clear_tail<TYPE, DIM>(vu, it.key1 - p0, wave * 64 + lane, 256);
            lds_done();
            workgroup_barrier();
        }
        if (p0 + G::TT > all_first && odd_values<TYPE, DIM>(vu, here(lane))) {  // the same for all waves
            uint32_t *odd = reinterpret_cast<uint32_t *>(lds + G::ODD);
            workgroup_barrier();
            if (wave == 0) mark_odd<TYPE, DIM>(vu, odd, here(lane));
            lds_done();
            workgroup_barrier();
            w.spoil(odd, p0, here(lane));
            workgroup_barrier();
        }
        if constexpr (TYPE == kTypeQ8_0) {
            float top = 0.0f;  // (every wave comes to the same unit)
            for (int k = lane; k < G::TT * G::NB; k += 64)
                top = fmaxf(top, fabsf((float)reinterpret_cast<const _Float16 *>(vu + G::TT * G::RB)[k]));
            w.raise_unit(top, vu, lane);
            expand<DIM>(unit_at(i + 1), vu, wide, ldexpf(1.0f, 8 - w.ve), wave * 64 + lane);
            lds_done();
            workgroup_barrier();
        }
        if (p0 >= wave_last) continue;  // behind all of this wave's rows
        if (p0 + G::TT > first) {
            w.mask(p0, lane);
            w.tops();
        }
        w.follow();
        w.weights();
        // (behind the last tile: scores of whatever lies there, and not used)
        w.scores(unit_at(i + 1), TYPE == kTypeQ8_0 ? wide : nullptr, lane);
        if constexpr (TYPE == kTypeQ8_0) w.template values16<true>(wide + G::TILE16, wide + 2 * G::TILE16, lane);
        else w.values(vu, lane);
        w.tops();
    }
    w.finish();
    const int c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int r = mine + 16 * t + c;
        if (r >= it.n_rows) continue;
        if (it.part < 0) {
            float *o = a.out + row_at(a, it, h, r, DIM);
#pragma unroll
            for (int d = 0; d < G::ND; ++d) *reinterpret_cast<v4f *>(o + d * 16 + g * 4) = w.acc[t][d] / w.l[t];
        } else {
            const size_t ps = (size_t)(it.part + r) * a.kv.n_kv + h;
#pragma unroll
            for (int d = 0; d < G::ND; ++d) *reinterpret_cast<v4f *>(a.part + ps * DIM + d * 16 + g * 4) = w.acc[t][d];
            if (g == 0) {
                float *d = a.part + a.part_cap * DIM + 2 * ps;
                d[0] = w.m[t];
                d[1] = w.l[t];
            }
        }
    }
    __syncthreads();
}

template <int TYPE, int DIM>
__global__ __launch_bounds__(256, (Geo<TYPE, DIM>::WAVES)) void attn_kernel(const AttnArgs args) {
    using G = Geo<TYPE, DIM>;
    extern __shared__ __align__(16) uint8_t lds[];
    const PlanHeader *hd = reinterpret_cast<const PlanHeader *>(args.head);
    // (constant memory: scalar loads)
    const auto *items = (const __attribute__((address_space(4))) AttnItem *)(uintptr_t)(hd + 1);
    const long long all = args.work >= 0 ? args.work : (long long)hd->n_items * args.kv.n_kv;
    for (long long i = blockIdx.x; i < all; i += gridDim.x) {
        // The arguments and the wave's number anew for each item: what the four
        // ways below make of them would else be computed in front of this loop
        // for all of them, and be moved in and out of vector registers (measured:
        // 3 to 8 % of the many-row ways).
        auto *ka = (const __attribute__((address_space(4))) AttnArgs *)__builtin_amdgcn_kernarg_segment_ptr();
        uint32_t w0 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        asm volatile("" : "+s"(ka), "+s"(w0));
        const int wave = (int)w0, lane = here(threadIdx.x & 63);
        AttnArgs a;
        a.q = ka->q;
        a.out = ka->out;
        a.head = ka->head;
        a.part = ka->part;
        a.kv.base = ka->kv.base;
        a.kv.page_bytes = ka->kv.page_bytes;
        a.kv.head_bytes = ka->kv.head_bytes;
        a.kv.page_shift = ka->kv.page_shift;
        a.kv.n_kv = ka->kv.n_kv;
        a.scale = ka->scale;
        a.group = ka->group;
        a.part_cap = ka->part_cap;
        const int n_kv = a.kv.n_kv, h = (int)i % n_kv;
        const auto &from = items[(int)i / n_kv];
        AttnItem it;
        it.row0 = from.row0;
        it.n_rows = from.n_rows;
        it.key0 = from.key0;
        it.key1 = from.key1;
        it.page_at = from.page_at;
        it.causal = from.causal;
        it.part = from.part;
        Source s;
        s.pages = (const __attribute__((address_space(4))) int32_t *)(uintptr_t)(a.head + it.page_at);
        s.base = a.kv.base + (size_t)h * a.kv.head_bytes;
        s.page_bytes = a.kv.page_bytes;
        s.head_bytes = a.kv.head_bytes;
        s.v_off = (uint32_t)n_kv * a.kv.head_bytes;
        s.shift = a.kv.page_shift;
        s.last = (it.key1 - 1) >> a.kv.page_shift;
        if (it.n_rows <= 16) attend_few<TYPE, DIM, 1>(a, it, s, h, lds, wave, lane);
        else if (G::PAIR && it.n_rows <= 32) attend_few<TYPE, DIM, G::PAIR ? 2 : 1>(a, it, s, h, lds, wave, lane);
        else if (G::ONE && (G::RT == 1 || it.n_rows <= 64)) {
            if constexpr (G::ONE) attend_many<TYPE, DIM, 1>(a, it, s, h, lds, wave, lane);
        } else {
            if constexpr (G::RT > 1) attend_many<TYPE, DIM, G::RT>(a, it, s, h, lds, wave, lane);
        }
    }
}

// Rows with several pieces: a workgroup joins a row's partial results of one
// kv head, out = sum_i 2^(m_i - m) acc_i / sum_i 2^(m_i - m) l_i.  Its groups of
// DIM / 4 lanes take every GROUPS-th piece, in order, and are added up in order:
// the result does not depend on timing.  Bound by the latency of three dependent
// loads (the list, the maxima, the sums), so every piece's loads go out at once.
template <int DIM>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnArgs a) {
    constexpr int W = DIM / 4, GROUPS = 256 / W, kMost = 256;
    __shared__ float weight[kMost];
    __shared__ int piece[kMost];
    __shared__ float red[4];
    __shared__ v4f sums[GROUPS * W];
    const PlanHeader *hd = reinterpret_cast<const PlanHeader *>(a.head);
    const int tid = threadIdx.x, n_kv = a.kv.n_kv, grp = tid / W, e = tid % W * 4;
    const float *mls = a.part + a.part_cap * DIM;
    const long long all = a.joins >= 0 ? a.joins : (long long)hd->n_joined * n_kv;
    for (long long w = blockIdx.x; w < all; w += gridDim.x) {
        const int i = (int)(w / n_kv), h = (int)(w % n_kv);
        const int row = a.head[hd->join_rows + i];
        const int p0 = a.head[hd->join_at + i], p1 = a.head[hd->join_at + i + 1];
        float m = -INFINITY, l = 0.0f;
        v4f acc = {0, 0, 0, 0};
        for (int from = p0; from < p1; from += kMost) {  // (one round up to 256 pieces)
            const int n = min(kMost, p1 - from);
            float mi = -INFINITY, li = 0.0f;
            int ps = 0;
            if (tid < n) {
                ps = a.head[from + tid];
                const float2 ml = *reinterpret_cast<const float2 *>(mls + 2 * ((size_t)ps * n_kv + h));
                mi = ml.x;
                li = ml.y;
            }
            const float wm = wave_max(mi);
            __syncthreads();
            if ((tid & 63) == 0) red[tid >> 6] = wm;
            __syncthreads();
            const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
            const float c = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            // a piece behind the row's last position is left out; others count with any weight, zero too (NaN)
            const bool out = mi == -INFINITY && li == 0.0f;
            const float f = out ? -1.0f : __builtin_amdgcn_exp2f(mi - mn);
            weight[tid] = f;
            piece[tid] = ps;
            m = mn;
            l *= c;
            acc *= c;
            __syncthreads();
            li = out ? 0.0f : f * li;
            li = wave_sum_f32(li);
            __syncthreads();
            if ((tid & 63) == 0) red[tid >> 6] = li;
            if (grp < GROUPS) {
#pragma unroll 4
                for (int p = grp; p < n; p += GROUPS) {
                    const float wp = weight[p];
                    const v4f v = *reinterpret_cast<const v4f *>(a.part + ((size_t)piece[p] * n_kv + h) * DIM + e);
                    if (!(wp < 0.0f)) acc += wp * v;
                }
            }
            __syncthreads();
            l += (red[0] + red[1]) + (red[2] + red[3]);
        }
        if (grp < GROUPS) sums[grp * W + tid % W] = acc;
        __syncthreads();
        if (tid < W) {
            v4f o = sums[tid];
#pragma unroll
            for (int k = 1; k < GROUPS; ++k) o += sums[k * W + tid];
            const PlanToken *pt = reinterpret_cast<const PlanToken *>(a.head) - (row / a.group + 1);
            *reinterpret_cast<v4f *>(a.out + (((size_t)pt->order * n_kv + h) * a.group + row % a.group) * DIM + e) = o / l;
        }
        __syncthreads();
    }
}

namespace {

template <int DIM>
int per_cu(int type) {
    return type == kTypeF32 ? Geo<kTypeF32, DIM>::PER_CU : type == kTypeF16 ? Geo<kTypeF16, DIM>::PER_CU : Geo<kTypeQ8_0, DIM>::PER_CU;
}

template <int TYPE, int DIM>
hipError_t allow_lds() {
    constexpr int bytes = Geo<TYPE, DIM>::LDS_BYTES;
    static_assert(bytes <= 160 * 1024, "the rings fit the gfx950 LDS");
    return hipFuncSetAttribute(reinterpret_cast<const void *>(attn_kernel<TYPE, DIM>),
                               hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}
template <int DIM>
hipError_t allow_lds(int type) {
    return type == kTypeF32 ? allow_lds<kTypeF32, DIM>() : type == kTypeF16 ? allow_lds<kTypeF16, DIM>() : allow_lds<kTypeQ8_0, DIM>();
}

template <int TYPE, int DIM>
hipError_t launch_typed(const AttnArgs &a, unsigned grid, hipStream_t st) {
    constexpr int bytes = Geo<TYPE, DIM>::LDS_BYTES;
    hipLaunchKernelGGL((attn_kernel<TYPE, DIM>), dim3(grid), dim3(256), bytes, st, a);
    return hipGetLastError();
}

template <int DIM>
hipError_t launch_attention(const AttnArgs &a, int type, unsigned grid, unsigned join_grid, hipStream_t st) {
    hipError_t e;
    if (type == kTypeF32) e = launch_typed<kTypeF32, DIM>(a, grid, st);
    else if (type == kTypeF16) e = launch_typed<kTypeF16, DIM>(a, grid, st);
    else e = launch_typed<kTypeQ8_0, DIM>(a, grid, st);
    if (e != hipSuccess) return e;
    if (join_grid != 0) hipLaunchKernelGGL((attn_join_kernel<DIM>), dim3(join_grid), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace

hipError_t attn_prepare(int type, int dim) {
    return dim == 64 ? allow_lds<64>(type) : dim == 96 ? allow_lds<96>(type) : dim == 128 ? allow_lds<128>(type) : allow_lds<256>(type);
}

int attn_workgroups(int type, int dim) {
    return 256 * (dim == 64 ? per_cu<64>(type) : dim == 96 ? per_cu<96>(type) : dim == 128 ? per_cu<128>(type) : per_cu<256>(type));
}

}  // namespace exq

using namespace exq;

extern "C" int edgexpu_hip_attention_dev(float *out, const float *q, edgexpu_hip_batch *b, int layer, float scale,
                                         void *stream) {
    if (!lib_ready("attention")) return 0;
    bool capturing = false;
    if (!batch_ready(b, layer, (hipStream_t)stream, "attention", &capturing)) return 0;
    if (b->plan.tokens.empty()) return 1;
    if (out == nullptr || q == nullptr || (((uintptr_t)out | (uintptr_t)q) & 15u) != 0 || !(fabsf(scale) < INFINITY)) {
        lib_error(-2, "attention: null buffer, q or out not 16-byte aligned, or scale %g not finite", (double)scale);
        return 0;
    }
    if (capturing) batch_recorded(b);
    const edgexpu_hip_kv *kv = b->kv;
    AttnArgs a = {};
    a.q = q;
    a.out = out;
    a.head = b->head();
    a.part = b->part;
    a.part_cap = b->part_cap;
    a.kv = kv_view(kv, layer);
    a.scale = scale;
    a.group = b->n_heads / kv->n_kv;
    // One workgroup an item and kv head; a captured call, whose plan may be
    // replaced before a replay, takes a fixed grid that walks whatever is there.
    const long long items = (long long)b->plan.items.size() * kv->n_kv;
    const long long joins = (long long)b->plan.join_rows.size() * kv->n_kv;
    a.work = capturing ? -1 : items;
    a.joins = capturing ? -1 : joins;
    const unsigned grid = capturing ? 1024u : (unsigned)std::min<long long>(items, 1 << 20);
    const unsigned join_grid = capturing ? 1024u : (unsigned)std::min<long long>(joins, 1 << 20);
    hipError_t e;
    switch (kv->dim) {
        case 64: e = launch_attention<64>(a, kv->type, grid, join_grid, (hipStream_t)stream); break;
        case 96: e = launch_attention<96>(a, kv->type, grid, join_grid, (hipStream_t)stream); break;
        case 128: e = launch_attention<128>(a, kv->type, grid, join_grid, (hipStream_t)stream); break;
        default: e = launch_attention<256>(a, kv->type, grid, join_grid, (hipStream_t)stream); break;
    }
    return lib_hip(e, "attention") ? 1 : 0;
}
