// Weight rows of each format as operands of the integer matrix cores, for the
// products with routed experts, and the packed activation they meet.
//
// A step of every product is a group of 256 elements of 16 weight rows against
// 16 tokens.  Operands of v_mfma_i32_16x16x64_i8: lane l supplies row l % 16 of A
// (a weight row) and column l % 16 of B (a token), 16 bytes of group g = l / 16;
// the 64 places of K may be any 64 elements as long as A and B agree.
// Accumulator register r of lane l is C[4 g + r][l % 16] = C[row][token].
//
// K-quants: sum_j sc_j sum_i q_i x_i over the sub-blocks j of a group has to be
// exact.  One product a sub-block, its sum times sc_j on the VALU, costs 8 (Q6_K:
// 16, K = 32 holding two) multiply-adds for each of a lane's 4 sums, more
// than the matrix cores' own time.  Here the scale goes into the operand instead:
// sc is cut into digits of base 8, sc = s0 + 8 s1 (+ 64 s2), and q * s fits 8 bits,
// so 4 products a digit sum a whole group and
//   sum = S0 + 8 S1 (+ 64 S2)
// costs one shift-add a digit.  q * s is one 16-bit packed product for four codes
// (each byte's product stays below 256, so none carries into the next):
//   Q4_K  15 * 7 = 105;  Q5_K  31 * 7 = 217, which is s8 - 128 with its top bit
//   turned, and 128 (1 + 8) sum x is added back;  Q6_K has signed scales and codes
//   of 6 bits, digits -3 .. 4 and the code less 32: -128 .. 124, even and odd codes
//   apart.
// The minima's sum, sum_j m_j sum_(i in j) x_i, is one product of f16 (integers
// below 2^11, exact, as is the sum below 2^24) with the tokens' 16-element sums.
//
// Blocks of 32 with one f16 scale (Q8_0, Q4_0, Q5_0): v_mfma_i32_16x16x32_i8 a
// block, then acc += S * (dw dx).
//
// Packed activation: a record of kMoeRec bytes for a token's group:
//   K-quants  int8 codes[256] | f16 sums of 16 elements [16] | f32 dx | i32 sum of all
//   others    int8 codes[256] | f32 dx[8] (a last group's missing blocks are zeros)
// 304 bytes: 16-byte aligned, and 8 records apart by 48 (mod 128), so that 16 lanes
// reading one place of 16 records from LDS meet no bank twice.
#pragma once

#include <hip/hip_runtime.h>

#include "common.h"
#include "formats.h"
#include "q8k.h"

namespace exq {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef short i16x2 __attribute__((ext_vector_type(2)));

constexpr int kMoeRec = 304, kMoeBs = 256, kMoeDx = 288, kMoeSum = 292;

__device__ __forceinline__ v4i mfma64(v4i a, v4i b, v4i c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v4i mfma32(long a, long b) {
    return __builtin_amdgcn_mfma_i32_16x16x32_i8(a, b, v4i{0, 0, 0, 0}, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma_f16(v4h a, v4h b) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, v4f{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
}
__device__ __forceinline__ long two_words(uint32_t lo, uint32_t hi) {
    return (long)((uint64_t)lo | ((uint64_t)hi << 32));
}
__device__ __forceinline__ uint32_t mul_u16x2(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(u16x2, a) * __builtin_bit_cast(u16x2, b));
}
__device__ __forceinline__ v4i as_v4i(const uint4 &v) { return v4i{(int)v.x, (int)v.y, (int)v.z, (int)v.w}; }

// ------------------------------------------------------------- activations

// A token's group of a K-quant product as the operand (lane: token l % 16, group g).
struct MoeXK {
    v4i c[4];
    v4h bs;
    float dx;
    int sum;
};
// ... of a product of 32-element blocks.
struct MoeX0 {
    long c[8];
    float dx[8];
};

// 16 lanes of a DPP row quantize 256 elements and write their record.  Lane 4 j + q
// holds elements 64 j + 8 q .. + 7 and 64 j + 32 + 8 q .. + 7 in xs.
__device__ __forceinline__ void moe_pack_k(const float (&xs)[16], int r, uint8_t *rec) {
    const int j = r >> 2, q = r & 3;
    int qv[16];
    const Q8KRow16 k = q8k_quantize_row16(xs, qv);
    uint32_t w[4];
    int sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = (uint32_t)(qv[4 * i] & 0xff) | ((uint32_t)(qv[4 * i + 1] & 0xff) << 8) |
               ((uint32_t)(qv[4 * i + 2] & 0xff) << 16) | ((uint32_t)qv[4 * i + 3] << 24);
        sum += (qv[4 * i] + qv[4 * i + 1]) + (qv[4 * i + 2] + qv[4 * i + 3]);
    }
    sum += (int)dpp_u32<kDppXor1>((uint32_t)sum);
    sum += (int)dpp_u32<kDppXor2>((uint32_t)sum);
    sum += (int)dpp_u32<kDppHalfMirror>((uint32_t)sum);
    sum += (int)dpp_u32<kDppMirror>((uint32_t)sum);
    *reinterpret_cast<uint2 *>(rec + 64 * j + 8 * q) = make_uint2(w[0], w[1]);
    *reinterpret_cast<uint2 *>(rec + 64 * j + 32 + 8 * q) = make_uint2(w[2], w[3]);
    if (q == 0) {
        const v4h b = {(_Float16)(float)k.lo, (_Float16)(float)k.lo_next, (_Float16)(float)k.hi,
                       (_Float16)(float)k.hi_next};
        *reinterpret_cast<v4h *>(rec + kMoeBs + 8 * j) = b;
    }
    if (r == 0) {
        *reinterpret_cast<float *>(rec + kMoeDx) = k.d;
        *reinterpret_cast<int *>(rec + kMoeSum) = sum;
    }
}

// 4 lanes quantize a block of 32 as quantize_q8_0_kernel does, lane g its elements
// 8 g .. + 7, and write them to block b (0..7) of the record.
__device__ __forceinline__ void moe_pack_0(const float (&a)[8], int b, int g, uint8_t *rec) {
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(a[i]));
    amax = fmaxf(amax, __uint_as_float(dpp_u32<kDppXor1>(__float_as_uint(amax))));
    amax = fmaxf(amax, __uint_as_float(dpp_u32<kDppXor2>(__float_as_uint(amax))));
    const float id = amax != 0.0f ? 127.0f / amax : 0.0f;
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = rintf(a[i] * id);
        const int k = (v >= -2147483648.0f && v < 2147483648.0f) ? (int)v : INT32_MIN;
        const int c = k < -128 ? -128 : (k > 127 ? 127 : k);
        w[i >> 2] |= (uint32_t)(c & 0xff) << (8 * (i & 3));
    }
    *reinterpret_cast<uint2 *>(rec + 32 * b + 8 * g) = make_uint2(w[0], w[1]);
    if (g == 0) *reinterpret_cast<float *>(rec + kMoeBs + 4 * b) = f16_bits_to_f32(f32_to_f16_rne(amax / 127.0f));
}

__device__ __forceinline__ void load_f8(const float *p, float *v) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

// Part `part` of a row's packing: K-quants 16 lanes a group of 256, others 32 lanes
// (4 a block).  x is the row, rec its first record, n its elements.
template <bool K>
__device__ __forceinline__ void moe_read_part(float (&v)[K ? 16 : 8], const float *x, int n, int part) {
    if (K) {
        const float *p = x + (size_t)(part >> 4) * kQKK + 64 * ((part & 15) >> 2) + 8 * (part & 3);
        load_f8(p, v);
        load_f8(p + 32, v + (K ? 8 : 0));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        if ((part >> 2) * 32 < n) load_f8(x + 8 * (size_t)part, v);
    }
}
template <bool K>
__device__ __forceinline__ void moe_put_part(const float (&v)[K ? 16 : 8], int part, uint8_t *rec) {
    if constexpr (K)
        moe_pack_k(v, part & 15, rec + (size_t)(part >> 4) * kMoeRec);
    else
        moe_pack_0(v, (part >> 2) & 7, part & 3, rec + (size_t)(part >> 5) * kMoeRec);
}
template <bool K>
__device__ __forceinline__ void moe_pack_part(const float *x, int n, int part, uint8_t *rec) {
    float v[K ? 16 : 8];
    moe_read_part<K>(v, x, n, part);
    moe_put_part<K>(v, part, rec);
}
__host__ __device__ constexpr int moe_groups(int n) { return (n + kQKK - 1) / kQKK; }
template <bool K>
__host__ __device__ constexpr int moe_pack_parts(int n) {
    return moe_groups(n) * (K ? 16 : 32);
}

// ---------------------------------------------------------------- K-quants
//
// W: raw registers of a group of the lane's row; Op: the operand; chunk(s, g): which
// 16 elements of the group lane group g holds in product s of 4; kLong: decode() is.

// A group's integer sums, a digit each, and the minima's.
template <class F>
struct MoeSums {
    v4i s[F::kDigits];
    v4f mn;
    float dx;
    int sum;
};
template <class F>
__device__ __forceinline__ void moe_mul_k(MoeSums<F> &m, const typename F::Op &o, const MoeXK &x) {
#pragma unroll
    for (int k = 0; k < F::kDigits; ++k) m.s[k] = v4i{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < F::kDigits; ++k) m.s[k] = mfma64(o.a[k][i], x.c[i], m.s[k]);
    if (F::kMin) m.mn = mfma_f16(o.mn, x.bs);
    m.dx = x.dx;
    m.sum = x.sum;
}
// acc += dx * (sum * d - minima * dmin)
template <class F>
__device__ __forceinline__ void moe_add_k(float (&acc)[4], const MoeSums<F> &m, const float (&d)[4],
                                          const float (&nd)[4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        int t = m.s[F::kDigits - 1][r];
#pragma unroll
        for (int k = F::kDigits - 2; k >= 0; --k) t = (t << 3) + m.s[k][r];
        if (F::kTurned) t += 1152 * m.sum;
        float v = (float)t * d[r];
        if (F::kMin) v = __builtin_fmaf(m.mn[r], nd[r], v);
        acc[r] = __builtin_fmaf(v, m.dx, acc[r]);
    }
}

template <class F>
__device__ __forceinline__ void moe_load_xk(MoeXK &x, const uint8_t *rec, int g) {
#pragma unroll
    for (int s = 0; s < 4; ++s) x.c[s] = as_v4i(*reinterpret_cast<const uint4 *>(rec + 16 * F::chunk(s, g)));
    x.bs = *reinterpret_cast<const v4h *>(rec + kMoeBs + 8 * g);
    const uint2 e = *reinterpret_cast<const uint2 *>(rec + kMoeDx);
    x.dx = __uint_as_float(e.x);
    x.sum = (int)e.y;
}

// d and -dmin of the rows 4 g + r, which the lane's sums belong to, from the word
// (d, dmin) that lane r16 of each group holds for its row.
__device__ __forceinline__ void moe_row_scales(uint32_t own, int g, float (&d)[4], float (&nd)[4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const uint32_t v = (uint32_t)__shfl((int)own, 4 * g + r, 64);
        d[r] = f16_bits_to_f32(v & 0xffffu);
        nd[r] = -f16_bits_to_f32(v >> 16);
    }
}

// The six-bit scales and minima of get_scale_min_k4 (src/gguf_quant.c:212-220), four a word.
struct SixBits {
    uint32_t s[2], m[2];
};
__device__ __forceinline__ SixBits six_bits(const uint4 &hd) {
    SixBits b;
    b.s[0] = hd.y & 0x3f3f3f3fu;
    b.s[1] = (hd.w & 0x0f0f0f0fu) | ((hd.y >> 2) & 0x30303030u);
    b.m[0] = hd.z & 0x3f3f3f3fu;
    b.m[1] = ((hd.w >> 4) & 0x0f0f0f0fu) | ((hd.z >> 2) & 0x30303030u);
    return b;
}
// The digits of four scales at once, and one of them in both halves of a word: byte
// 2 (g / 2) + h is the chunk's h-th scale for lane group g.
struct Digits8 {
    uint32_t lo[2], hi[2];
};
__device__ __forceinline__ Digits8 digits8(const SixBits &b) {
    Digits8 d;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        d.lo[i] = b.s[i] & 0x07070707u;
        d.hi[i] = (b.s[i] >> 3) & 0x07070707u;
    }
    return d;
}
__device__ __forceinline__ uint32_t both_halves(uint32_t bytes, int g, int h) {
    return __builtin_amdgcn_perm(0u, bytes, 0x0c000c00u + 0x00010001u * (uint32_t)(2 * (g >> 1) + h));
}
// Minima of lane group g's four 16-element sums.
__device__ __forceinline__ v4h min_operand(const SixBits &b, int g) {
    // a byte below 0x64 is the f16 1024 + m
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const uint32_t w = (g & 2) ? b.m[1] : b.m[0];
    const uint32_t sel = 0x04000400u + 0x00010001u * (uint32_t)(2 * (g & 1));
    const h2 k = {(_Float16)1024.0f, (_Float16)1024.0f};
    const h2 x = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, sel)) - k;
    const h2 y = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, sel + 0x00010001u)) - k;
    return v4h{x[0], x[1], y[0], y[1]};
}

struct MoeQ4K {
    static constexpr bool kK = true, kMin = true, kTurned = false;
    static constexpr int kType = kTypeQ4_K, kDigits = 2, kBytes = kBytesQ4_K;
    static constexpr bool kLong = false;
    struct W {
        uint4 hd, q[2];
    };
    struct Op {
        v4i a[2][4];
        v4h mn;
        uint32_t dm;
    };
    typedef MoeXK X;
    __device__ static constexpr int chunk(int s, int g) { return 8 * (s >> 1) + 4 * (g >> 1) + 2 * (s & 1) + (g & 1); }
    __device__ static __forceinline__ void load_w(W &w, const uint8_t *row, int u, int, int g) {
        const uint8_t *p = row + (size_t)u * kBytes;
        w.hd = *reinterpret_cast<const uint4 *>(p);
        w.q[0] = *reinterpret_cast<const uint4 *>(p + 16 + 16 * g);
        w.q[1] = *reinterpret_cast<const uint4 *>(p + 80 + 16 * g);
    }
    __device__ static __forceinline__ void decode(Op &o, const W &w, int g) {
        const SixBits b = six_bits(w.hd);
        const Digits8 dg = digits8(b);
        o.mn = min_operand(b, g);
        o.dm = w.hd.x;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t q[4] = {w.q[i].x, w.q[i].y, w.q[i].z, w.q[i].w};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t s0 = both_halves(dg.lo[i], g, h), s1 = both_halves(dg.hi[i], g, h);
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const uint32_t c = (q[v] >> (4 * h)) & 0x0f0f0f0fu;
                    o.a[0][2 * i + h][v] = (int)mul_u16x2(c, s0);
                    o.a[1][2 * i + h][v] = (int)mul_u16x2(c, s1);
                }
            }
        }
    }
};

struct MoeQ5K {
    static constexpr bool kK = true, kMin = true, kTurned = true;
    static constexpr int kType = kTypeQ5_K, kDigits = 2, kBytes = kBytesQ5_K;
    static constexpr bool kLong = false;
    struct W {
        uint4 hd, h, q[2];
    };
    typedef MoeQ4K::Op Op;
    typedef MoeXK X;
    __device__ static constexpr int chunk(int s, int g) { return MoeQ4K::chunk(s, g); }
    __device__ static __forceinline__ void load_w(W &w, const uint8_t *row, int u, int, int g) {
        const uint8_t *p = row + (size_t)u * kBytes;
        w.hd = *reinterpret_cast<const uint4 *>(p);
        w.h = *reinterpret_cast<const uint4 *>(p + 16 + 16 * (g & 1));
        w.q[0] = *reinterpret_cast<const uint4 *>(p + 48 + 16 * g);
        w.q[1] = *reinterpret_cast<const uint4 *>(p + 112 + 16 * g);
    }
    __device__ static __forceinline__ void decode(Op &o, const W &w, int g) {
        const SixBits b = six_bits(w.hd);
        const Digits8 dg = digits8(b);
        o.mn = min_operand(b, g);
        o.dm = w.hd.x;
        const uint32_t fifth[4] = {w.h.x, w.h.y, w.h.z, w.h.w};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t q[4] = {w.q[i].x, w.q[i].y, w.q[i].z, w.q[i].w};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t s0 = both_halves(dg.lo[i], g, h), s1 = both_halves(dg.hi[i], g, h);
                const int bit = 4 * i + 2 * (g >> 1) + h;  // of the 64-element chunk 2 i + g / 2, half h
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const uint32_t c = ((q[v] >> (4 * h)) & 0x0f0f0f0fu) | (((fifth[v] >> bit) & 0x01010101u) << 4);
                    o.a[0][2 * i + h][v] = (int)(mul_u16x2(c, s0) ^ 0x80808080u);
                    o.a[1][2 * i + h][v] = (int)(mul_u16x2(c, s1) ^ 0x80808080u);
                }
            }
        }
    }
};

// 16 bytes from byte sh = 0 or 2 of five words on.  Wide loads at 2 mod 4 run several times slower
// (ldg16_a2), so that words are read from the 4-byte address below.
__device__ __forceinline__ void join_even(uint32_t (&v)[4], const uint4 &w, uint32_t end, uint32_t sh) {
    v[0] = __builtin_amdgcn_alignbyte(w.y, w.x, sh);
    v[1] = __builtin_amdgcn_alignbyte(w.z, w.y, sh);
    v[2] = __builtin_amdgcn_alignbyte(w.w, w.z, sh);
    v[3] = __builtin_amdgcn_alignbyte(end, w.w, sh);
}

struct MoeQ6K {
    static constexpr bool kK = true, kMin = false, kTurned = false;
    static constexpr int kType = kTypeQ6_K, kDigits = 3, kBytes = kBytesQ6_K;
    static constexpr bool kLong = true;
    struct W {
        uint4 l[2], h[2], sc;  // as words from the 4-byte address below; the scales are the same in all lane groups
        uint32_t d, sh;        // the block's last word: two scales, then d
    };
    struct Op {
        v4i a[3][4];
        v4h mn;
        uint32_t dm;
    };
    typedef MoeXK X;
    __device__ static constexpr int chunk(int s, int g) { return 4 * s + g; }
    __device__ static __forceinline__ void load_w(W &w, const uint8_t *row, int u, int, int g) {
        const uint8_t *p = row + (size_t)u * kBytes;
        // (where it begins: the aligned word that holds d may end behind the tensor)
        __builtin_memcpy(&w.d, p + kBytes - 4, 4);
        w.sh = (uint32_t)((uintptr_t)p & 3u);
        p -= w.sh;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            w.l[i] = *reinterpret_cast<const uint4 *>(p + 64 * i + 16 * g);
            w.h[i] = *reinterpret_cast<const uint4 *>(p + 128 + 32 * i + 16 * (g & 1));
        }
        w.sc = *reinterpret_cast<const uint4 *>(p + 192);
    }
    __device__ static __forceinline__ void decode(Op &o, const W &w, int g) {
        o.dm = w.d >> 16;
        o.mn = v4h{0, 0, 0, 0};
        uint32_t sc[4];
        join_even(sc, w.sc, w.d, w.sh);  // (of the last word only where sh is 2: it begins at the fifth word then)
        // A piece's fifth word is the next piece's first: lane group g + 1's, or the next run's in group 0 (or,
        // of two groups, in the even one), and behind the last the scales'.  Loads of two bytes for them cost
        // a wave as much as whole ones.
        const int lane = __lane_id(), next = ((lane + 16) & 63) << 2, other = (lane ^ 16) << 2;
        const uint32_t end_l[2] = {
            (uint32_t)__builtin_amdgcn_ds_bpermute(next, (int)(g == 0 ? w.l[1].x : w.l[0].x)),
            (uint32_t)__builtin_amdgcn_ds_bpermute(next, (int)(g == 0 ? w.h[0].x : w.l[1].x))};
        const uint32_t over = (uint32_t)__builtin_amdgcn_ds_bpermute(other, (int)w.h[1].x);
        const uint32_t end_h[2] = {
            (uint32_t)__builtin_amdgcn_ds_bpermute(other, (int)((g & 1) ? w.h[0].x : w.h[1].x)),
            (g & 1) ? w.sc.x : over};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t l[4], hh[4];
            join_even(l, w.l[i], end_l[i], w.sh);
            join_even(hh, w.h[i], end_h[i], w.sh);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int q = (int)(int8_t)(sc[2 * i + h] >> (8 * g));  // scale 8 i + 4 h + g
                const int s0 = ((q + 3) & 7) - 3, r1 = (q - s0) >> 3, s1 = ((r1 + 3) & 7) - 3, s2 = (r1 - s1) >> 3;
                const int dig[3] = {s0, s1, s2};
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    // this half's two high bits are bits 2 (g / 2) + 4 h of each byte
                    const uint32_t top = (hh[v] >> (2 * (g >> 1) + 4 * h)) & 0x03030303u;
                    const uint32_t c = ((l[v] >> (4 * h)) & 0x0f0f0f0fu) | (top << 4);
                    const i16x2 even = __builtin_bit_cast(i16x2, c & 0x00ff00ffu) - (short)32;
                    const i16x2 odd = __builtin_bit_cast(i16x2, (c >> 8) & 0x00ff00ffu) - (short)32;
#pragma unroll
                    for (int k = 0; k < 3; ++k) {
                        const short s = (short)dig[k];
                        o.a[k][2 * i + h][v] = (int)__builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, odd * s),
                                                                          __builtin_bit_cast(uint32_t, even * s),
                                                                          0x06020400u);
                    }
                }
            }
        }
    }
};

// ------------------------------------------------------- blocks of 32 elements
//
// A row of n blocks; those past the end of a last group are not read (their
// codes and scales are zeros).

// Scales of the rows 4 g + r for the group's 8 blocks, from the word (blocks g, g + 4)
// that lane r16 of group g holds for its row.
__device__ __forceinline__ void moe_block_scales(uint32_t own, int g, float (&d)[8][4]) {
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t v = (uint32_t)__shfl((int)own, 16 * b + 4 * g + r, 64);
            d[b][r] = f16_bits_to_f32(v & 0xffffu);
            d[b + 4][r] = f16_bits_to_f32(v >> 16);
        }
}

struct MoeOp0 {
    long a[8];
    uint32_t dm;
};

__device__ __forceinline__ void moe_dot_0(float (&acc)[4], const MoeOp0 &o, const MoeX0 &x, const float (&d)[8][4]) {
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        const v4i s = mfma32(o.a[b], x.c[b]);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] = __builtin_fmaf((float)s[r], d[b][r] * x.dx[b], acc[r]);
    }
}

template <class F>
__device__ __forceinline__ void moe_load_x0(MoeX0 &x, const uint8_t *rec, int g) {
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        const uint2 v = F::kQ80 ? *reinterpret_cast<const uint2 *>(rec + 32 * b + 8 * (((g & 1) << 1) | (g >> 1)))
                                : make_uint2(*reinterpret_cast<const uint32_t *>(rec + 32 * b + 4 * g),
                                             *reinterpret_cast<const uint32_t *>(rec + 32 * b + 16 + 4 * g));
        x.c[b] = two_words(v.x, v.y);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float4 d = *reinterpret_cast<const float4 *>(rec + kMoeBs + 16 * i);
        x.dx[4 * i] = d.x, x.dx[4 * i + 1] = d.y, x.dx[4 * i + 2] = d.z, x.dx[4 * i + 3] = d.w;
    }
}

// Scales of blocks g and g + 4 of group u.
template <int BYTES>
__device__ __forceinline__ uint32_t load_scales(const uint8_t *row, int u, int n, int g) {
    const int b0 = 8 * u + g, b1 = b0 + 4;
    const uint32_t lo = b0 < n ? *reinterpret_cast<const uint16_t *>(row + (size_t)b0 * BYTES) : 0u;
    const uint32_t hi = b1 < n ? *reinterpret_cast<const uint16_t *>(row + (size_t)b1 * BYTES) : 0u;
    return lo | (hi << 16);
}

// Lane groups 0 and 1 read the halves of a pair's even block, 2 and 3 those of the
// odd one; v_permlane32_swap then leaves group g with the 8-byte piece {0, 2, 1, 3}[g] of
// either block.
struct MoeQ80 {
    static constexpr bool kK = false, kQ80 = true;
    static constexpr int kType = kTypeQ8_0, kBytes = kBytesQ8_0;
    static constexpr bool kLong = true;
    struct W {
        uint4 q[4];
        uint32_t d;
    };
    typedef MoeOp0 Op;
    typedef MoeX0 X;
    __device__ static __forceinline__ void load_w(W &w, const uint8_t *row, int u, int n, int g) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int b = 8 * u + 2 * i + (g >> 1);
            w.q[i] = ldg16_a2(row + (size_t)min(b, n - 1) * kBytes + 2 + 16 * (g & 1));
        }
        w.d = load_scales<kBytes>(row, u, n, g);
    }
    __device__ static __forceinline__ void decode(Op &o, const W &w, int) {
        o.dm = w.d;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const auto x = __builtin_amdgcn_permlane32_swap(w.q[i].x, w.q[i].z, false, false);
            const auto y = __builtin_amdgcn_permlane32_swap(w.q[i].y, w.q[i].w, false, false);
            o.a[2 * i] = two_words((uint32_t)x[0], (uint32_t)y[0]);
            o.a[2 * i + 1] = two_words((uint32_t)x[1], (uint32_t)y[1]);
        }
    }
};

// Lane group g holds elements 4 g .. + 3 and 16 + 4 g .. + 3 of a block: the low and
// high nibbles of one word of its codes, less 8 (Q5_0, with their fifth bits, less 16).
__device__ __forceinline__ uint32_t less_each(uint32_t c, uint32_t bias) {
    // (a code is below 128: 0x80 + c - bias borrows nothing, and its top bit turned is the sign)
    return ((c | 0x80808080u) - bias) ^ 0x80808080u;
}
struct MoeQ40 {
    static constexpr bool kK = false, kQ80 = false;
    static constexpr int kType = kTypeQ4_0, kBytes = kBytesQ4_0;
    static constexpr bool kLong = true;
    struct W {
        uint32_t q[8], d;
    };
    typedef MoeOp0 Op;
    typedef MoeX0 X;
    __device__ static __forceinline__ void load_w(W &w, const uint8_t *row, int u, int n, int g) {
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const uint8_t *p = row + (size_t)min(8 * u + b, n - 1) * kBytes + 2 + 4 * g;
            w.q[b] = (uint32_t)*reinterpret_cast<const uint16_t *>(p) |
                     ((uint32_t)*reinterpret_cast<const uint16_t *>(p + 2) << 16);
        }
        w.d = load_scales<kBytes>(row, u, n, g);
    }
    __device__ static __forceinline__ void decode(Op &o, const W &w, int) {
        o.dm = w.d;
#pragma unroll
        for (int b = 0; b < 8; ++b)
            o.a[b] = two_words(less_each(w.q[b] & 0x0f0f0f0fu, 0x08080808u),
                               less_each((w.q[b] >> 4) & 0x0f0f0f0fu, 0x08080808u));
    }
};

struct MoeQ50 {
    static constexpr bool kK = false, kQ80 = false;
    static constexpr int kType = kTypeQ5_0, kBytes = kBytesQ5_0;
    static constexpr bool kLong = true;
    struct W {
        uint32_t q[8], h[8], d;
    };
    typedef MoeOp0 Op;
    typedef MoeX0 X;
    __device__ static __forceinline__ void load_w(W &w, const uint8_t *row, int u, int n, int g) {
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const uint8_t *p = row + (size_t)min(8 * u + b, n - 1) * kBytes;
            w.h[b] = (uint32_t)*reinterpret_cast<const uint16_t *>(p + 2) |
                     ((uint32_t)*reinterpret_cast<const uint16_t *>(p + 4) << 16);
            w.q[b] = (uint32_t)*reinterpret_cast<const uint16_t *>(p + 6 + 4 * g) |
                     ((uint32_t)*reinterpret_cast<const uint16_t *>(p + 8 + 4 * g) << 16);
        }
        w.d = load_scales<kBytes>(row, u, n, g);
    }
    __device__ static __forceinline__ void decode(Op &o, const W &w, int g) {
        o.dm = w.d;
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const uint32_t lo = (w.q[b] & 0x0f0f0f0fu) | spread4_bit4((w.h[b] >> (4 * g)) & 15u);
            const uint32_t hi = ((w.q[b] >> 4) & 0x0f0f0f0fu) | spread4_bit4((w.h[b] >> (16 + 4 * g)) & 15u);
            o.a[b] = two_words(less_each(lo, 0x10101010u), less_each(hi, 0x10101010u));
        }
    }
};

// ------------------------------------------------------------------ both kinds

// The operand made where it stands, in its own registers: the raw registers are then free
// for the next loads.  Left to the compiler the decoding moves down to the products, the loads
// go to other registers, and the copies between the two wait for every load in flight.
__device__ __forceinline__ void moe_hold(v4i (&a)[4]) {
    asm volatile("" : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]), "+v"(a[3]));
}
template <class Op>
__device__ __forceinline__ void moe_hold_op(Op &o) {
    if constexpr (sizeof(o.a) == sizeof(long[8])) {
        asm volatile("" : "+v"(o.a[0]), "+v"(o.a[1]), "+v"(o.a[2]), "+v"(o.a[3]), "+v"(o.a[4]), "+v"(o.a[5]),
                     "+v"(o.a[6]), "+v"(o.a[7]), "+v"(o.dm));
    } else {
#pragma unroll
        for (auto &digit : o.a) moe_hold(digit);
        asm volatile("" : "+v"(o.dm), "+v"(o.mn));
    }
}

// The rows' scales of a lane's sums.
template <class F, bool K = F::kK>
struct MoeScales {
    float d[4], nd[4];
    __device__ __forceinline__ void from(const typename F::Op &o, int g) { moe_row_scales(o.dm, g, d, nd); }
    __device__ __forceinline__ void dot(float (&acc)[4], const typename F::Op &o, const MoeXK &x) const {
        MoeSums<F> m;
        moe_mul_k<F>(m, o, x);
        moe_add_k<F>(acc, m, d, nd);
    }
};
template <class F>
struct MoeScales<F, false> {
    float d[8][4];
    __device__ __forceinline__ void from(const typename F::Op &o, int g) { moe_block_scales(o.dm, g, d); }
    __device__ __forceinline__ void dot(float (&acc)[4], const typename F::Op &o, const MoeX0 &x) const {
        moe_dot_0(acc, o, x, d);
    }
};
template <class F>
__device__ __forceinline__ void moe_load_x(typename F::X &x, const uint8_t *rec, int g) {
    if constexpr (F::kK)
        moe_load_xk<F>(x, rec, g);
    else
        moe_load_x0<F>(x, rec, g);
}

}  // namespace exq
