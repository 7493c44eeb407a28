// Per-head RMSNorm and position rotation of queries and keys in one pass, with
// the key/value cache write (the reference runs them one after the other:
// RMSNorm, RoPE in its two pairings, among src/cpu_kernel.c:200-460 and
// :659-972, and a copy into the cache window, src/kv_cache.c:22-127).
//
//   y = x * (1 / sqrt(mean(x^2) + eps)) * w         squares summed in double
//   (a, b) -> (a cos - b sin, a sin + b cos)        angle = pos * scale * base^(-2i/n_rot) / factor_i
//
// The angle is kept in turns in 64 bits (pos * turns_i) and its whole turns
// are taken off there, so a position of 10^5 has the same accuracy as one of
// 10.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <new>

#include "kv.h"
#include "lib.h"

struct edgexpu_hip_rope {
    int n_rot = 0, interleaved = 0;
    double *turns = nullptr;  // device, n_rot / 2
};

namespace exq {

struct RopeArgs {
    const float *q, *k, *v;
    long long ldq, ldk, ldv;
    float *q_out, *k_out;
    const float *qw, *kw;
    const double *turns;
    const int32_t *pos;   // by token; null: from the plan
    const int32_t *head;  // the plan; null without a cache
    KvView kv;
    float eps;
    int m, n_heads, n_kv, dim, n_rot, interleaved;
    int waves;  // of a token (rope_rows_kernel)
};

// The token of a call, its position and its slot.
struct RopeToken {
    int pos, slot;
};
__device__ __forceinline__ RopeToken rope_token(const RopeArgs &a, int t) {
    if (a.head != nullptr) {
        const PlanToken *pt = reinterpret_cast<const PlanToken *>(a.head) - (t + 1);
        return {pt->pos, pt->slot};
    }
    return {a.pos != nullptr ? a.pos[t] : 0, 0};
}

// A block's largest magnitude is the largest bit pattern: a NaN is above all, and
// makes the scale NaN (edgexpu_hip_quantize_q8_0_dev leaves it out of the maximum,
// and a cached NaN would be lost).  Else codes and scales are that quantizer's:
// codes by 127 / max, out of range -128, the scale max / 127 rounded to f16.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ int q8_code(float v, float id) {
    const float x = rintf(v * id);
    return fabsf(x) <= 127.0f ? (int)x : -128;
}

// Any head size, pairing and alignment.  TYPE: the cache's, -1: k goes to k_out.
// One wave a head of a token, in 64 bits; the row passes through LDS for its
// partners.
template <int TYPE>
__global__ __launch_bounds__(256) void rope_kernel(const RopeArgs a) {
    __shared__ double rows[4][256];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int slots = a.n_heads + a.n_kv * (TYPE >= 0 ? 2 : 1);
    const int m = a.head != nullptr && a.m < 0 ? reinterpret_cast<const PlanHeader *>(a.head)->n_tokens : a.m;
    const long long id = (long long)blockIdx.x * 4 + wave;
    const int t = (int)(id / slots), s = (int)(id % slots);
    const bool live = t < m;
    const bool is_q = s < a.n_heads, is_v = s >= a.n_heads + a.n_kv;
    const int h = is_q ? s : is_v ? s - a.n_heads - a.n_kv : s - a.n_heads;
    const float *w = is_q ? a.qw : is_v ? nullptr : a.kw;
    double z[4] = {0.0, 0.0, 0.0, 0.0};
    int pos = 0, slot = 0;
    if (live) {
        const RopeToken tok = rope_token(a, t);
        pos = tok.pos;
        slot = tok.slot;
        const float *x = is_q ? a.q + t * a.ldq : is_v ? a.v + t * a.ldv : a.k + t * a.ldk;
        x += (size_t)h * a.dim;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (lane + 64 * j < a.dim) z[j] = (double)x[lane + 64 * j];
    }
    if (w != nullptr) {  // (the same for the whole wave)
        double ss = 0.0;
#pragma unroll
        for (int j = 0; j < 4; ++j) ss += z[j] * z[j];
        const double scale = 1.0 / sqrt(wave_sum_f64(ss) / (double)a.dim + (double)a.eps);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (lane + 64 * j < a.dim) z[j] = z[j] * scale * (double)w[lane + 64 * j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) rows[wave][lane + 64 * j] = z[j];
    __syncthreads();
    if (!live) return;
    if (!is_v) {
        const int half = a.n_rot >> 1;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int e = lane + 64 * j;
            if (e >= a.n_rot) continue;
            const bool first = a.interleaved ? (e & 1) == 0 : e < half;
            const int i = a.interleaved ? e >> 1 : first ? e : e - half;
            const int other = a.interleaved ? e ^ 1 : first ? e + half : e - half;
            double turn = (double)pos * a.turns[i];
            turn -= rint(turn);
            double sn, cs;
            sincospi(2.0 * turn, &sn, &cs);
            const double o = rows[wave][other];
            z[j] = first ? z[j] * cs - o * sn : o * sn + z[j] * cs;
        }
    }
    const float y[4] = {(float)z[0], (float)z[1], (float)z[2], (float)z[3]};
    if (is_q || TYPE < 0) {
        float *out = (is_q ? a.q_out + ((size_t)t * a.n_heads + h) * a.dim : a.k_out + ((size_t)t * a.n_kv + h) * a.dim);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (lane + 64 * j < a.dim) out[lane + 64 * j] = y[j];
        return;
    }
    const int off = slot & ((1 << a.kv.page_shift) - 1);
    uint8_t *base = a.kv.base + (size_t)(slot >> a.kv.page_shift) * a.kv.page_bytes +
                    (size_t)((is_v ? a.n_kv : 0) + h) * a.kv.head_bytes;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int e = lane + 64 * j;
        if (TYPE == kTypeQ8_0) {
            uint32_t most = row16_max_u32(magnitude(y[j]));
            most = max(most, (uint32_t)__shfl_xor((int)most, 16, 64));
            if (e >= a.dim) continue;
            const float top = __uint_as_float(most), id = top != 0.0f ? 127.0f / top : 0.0f;
            reinterpret_cast<int8_t *>(base)[(size_t)off * a.dim + e] = (int8_t)q8_code(y[j], id);
            if ((lane & 31) == 0)
                reinterpret_cast<uint16_t *>(base + ((size_t)a.dim << a.kv.page_shift))[off * (a.dim / 32) + e / 32] =
                    (uint16_t)f32_to_f16_rne(top / 127.0f);
        } else if (e < a.dim) {
            if (TYPE == kTypeF16) reinterpret_cast<_Float16 *>(base)[(size_t)off * a.dim + e] = (_Float16)y[j];
            else reinterpret_cast<float *>(base)[(size_t)off * a.dim + e] = y[j];
        }
    }
}

// Heads of 64, 96, 128 or 256 values at 16-byte addresses.  LPH lanes hold a
// head, four neighbouring values each, so a wave does 64 / LPH heads at once
// with 16-byte loads, sums a head's squares over its lanes, and finds a value's
// partner in its own registers (interleaved) or in the lane half a rotation
// away.  A wave keeps one token: its sines and cosines are computed once for all
// its heads, kAhead of which are loaded at a time.  Bound by the bytes for many
// tokens (8192 tokens of 32 + 2 x 8 heads of 128 to f16: 369 MB in 75 us, 4.9
// TB/s; a head a wave with every value's sine of its own took 260) and by the
// chain plan -> position -> sine -> store for few (one token 3.5 us), where a
// token takes several waves.
//
// Q8_0 keys are normed and rotated in 64 bits: a code next to a border depends
// on the last bits of its value, and with them it is the code of the exact one.
template <int TYPE, int LPH>
__global__ __launch_bounds__(256) void rope_rows_kernel(const RopeArgs a) {
    typedef float v4f __attribute__((ext_vector_type(4)));
    constexpr int HPW = 64 / LPH, kAhead = 4;
    constexpr bool EXACT_K = TYPE == kTypeQ8_0;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int sub = lane / LPH, l = lane % LPH, e = 4 * l;
    const int m = a.head != nullptr && a.m < 0 ? reinterpret_cast<const PlanHeader *>(a.head)->n_tokens : a.m;
    const int qi = (a.n_heads + HPW - 1) / HPW, ki = (a.n_kv + HPW - 1) / HPW;  // steps of HPW heads
    const int steps = qi + ki * (TYPE >= 0 ? 2 : 1);
    const int id = (int)(blockIdx.x * 4 + wave), t = id / a.waves, part = id % a.waves;
    if (t >= m) return;
    const int s0 = (int)((long long)steps * part / a.waves), s1 = (int)((long long)steps * (part + 1) / a.waves);
    const bool here = e < a.dim;
    const RopeToken tok = rope_token(a, t);

    const auto row = [&](int s, int &h) -> const float * {  // this lane's head of a step and its row; null: none
        const bool q = s < qi, v = s >= qi + ki;
        h = (q ? s : v ? s - qi - ki : s - qi) * HPW + sub;
        if (h >= (q ? a.n_heads : a.n_kv) || !here) return nullptr;
        return (q ? a.q + (size_t)t * a.ldq : v ? a.v + (size_t)t * a.ldv : a.k + (size_t)t * a.ldk) + (size_t)h * a.dim + e;
    };
    v4f x[kAhead];
    const auto fetch = [&](int s) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            int h;
            const float *p = s + i < s1 ? row(s + i, h) : nullptr;
            x[i] = p != nullptr ? *reinterpret_cast<const v4f *>(p) : v4f{0, 0, 0, 0};
        }
    };
    fetch(s0);
    v4f wq = {1, 1, 1, 1}, wk = wq;
    if (a.qw != nullptr && here) wq = *reinterpret_cast<const v4f *>(a.qw + e);
    if (a.kw != nullptr && here) wk = *reinterpret_cast<const v4f *>(a.kw + e);
    // Sines and cosines of this lane's four values; the sign of the sine is the
    // value's place in its pair.  Two are computed here: interleaved, they serve
    // two values each; else the lane with the partners has the same four angles
    // and computes the other two.
    const int half = a.n_rot >> 1;
    const bool turns = e < a.n_rot, low = a.interleaved || e < half;
    const int other = (lane - l + (a.interleaved || !turns ? l : e < half ? l + half / 4 : l - half / 4)) * 4;
    const auto swap32 = [other](float v) { return __int_as_float(__builtin_amdgcn_ds_bpermute(other, __float_as_int(v))); };
    const auto swap64 = [other](double v) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute(other, (int)(uint32_t)b);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_bpermute(other, (int)(uint32_t)(b >> 32));
        return __builtin_bit_cast(double, (uint64_t)lo | (uint64_t)hi << 32);
    };
    float cs[4], sn[4];
    double csd[4], snd[4];
    const bool exact = EXACT_K && s0 < qi + ki && s1 > qi;  // the wave has keys
    {
        float c[2], n[2];
        double cd[2], nd[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = a.interleaved ? (e >> 1) + j : low ? e + j : e - half + 2 + j;
            double turn = turns ? (double)tok.pos * a.turns[i] : 0.0;
            turn -= rint(turn);
            if (EXACT_K && exact) {
                sincospi(2.0 * turn, &nd[j], &cd[j]);
                n[j] = (float)nd[j];
                c[j] = (float)cd[j];
            } else {
                sincospif(2.0f * (float)turn, &n[j], &c[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (a.interleaved) {
                cs[j] = c[j >> 1];
                sn[j] = j & 1 ? n[j >> 1] : -n[j >> 1];
                if (EXACT_K && exact) {
                    csd[j] = cd[j >> 1];
                    snd[j] = j & 1 ? nd[j >> 1] : -nd[j >> 1];
                }
                continue;
            }
            const float oc = swap32(c[j & 1]), on = swap32(n[j & 1]);
            const bool mine = (j < 2) == low;
            cs[j] = mine ? c[j & 1] : oc;
            sn[j] = mine ? n[j & 1] : on;
            sn[j] = low ? -sn[j] : sn[j];
            if (EXACT_K && exact) {
                const double ocd = swap64(cd[j & 1]), ond = swap64(nd[j & 1]);
                csd[j] = mine ? cd[j & 1] : ocd;
                snd[j] = mine ? nd[j & 1] : ond;
                snd[j] = low ? -snd[j] : snd[j];
            }
        }
    }
    const auto partner = [&](const float (&y)[4], int j) {
        if (a.interleaved) return y[j ^ 1];
        return swap32(y[j]);
    };
    const int off = tok.slot & ((1 << a.kv.page_shift) - 1);
    uint8_t *page = TYPE >= 0 ? a.kv.base + (size_t)(tok.slot >> a.kv.page_shift) * a.kv.page_bytes : nullptr;
    for (int s = s0; s < s1; s += kAhead) {
        v4f now[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) now[i] = x[i];
        if (s + kAhead < s1) fetch(s + kAhead);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (s + i >= s1) break;
            const bool is_q = s + i < qi, is_v = s + i >= qi + ki;
            float y[4] = {now[i][0], now[i][1], now[i][2], now[i][3]};
            if (!is_v) {
                const bool norm = (is_q ? a.qw : a.kw) != nullptr;
                double ss = 0.0;
                if (norm) ss = wave_sum_f64<LPH>(square4(make_float4(y[0], y[1], y[2], y[3])));
                if (EXACT_K && !is_q) {
                    const double scale = norm ? 1.0 / sqrt(ss / (double)a.dim + (double)a.eps) : 1.0;
                    double z[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) z[j] = norm ? (double)y[j] * scale * (double)wk[j] : (double)y[j];
                    double o[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[j] = a.interleaved ? z[j ^ 1] : swap64(z[j]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[j] = (float)(turns ? fma(z[j], csd[j], o[j] * snd[j]) : z[j]);
                } else {
                    if (norm) {
                        const float scale = rms_scale(ss, a.dim, a.eps);
#pragma unroll
                        for (int j = 0; j < 4; ++j) y[j] = y[j] * scale * (is_q ? wq[j] : wk[j]);
                    }
                    if (half != 0) {
                        float o[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[j] = partner(y, j);
#pragma unroll
                        for (int j = 0; j < 4; ++j) y[j] = turns ? fmaf(y[j], cs[j], o[j] * sn[j]) : y[j];
                    }
                }
            }
            int h;
            const bool some = row(s + i, h) != nullptr;
            const v4f out = {y[0], y[1], y[2], y[3]};
            if (is_q || TYPE < 0) {
                float *o = is_q ? a.q_out + ((size_t)t * a.n_heads + h) * a.dim + e : a.k_out + ((size_t)t * a.n_kv + h) * a.dim + e;
                if (some) *reinterpret_cast<v4f *>(o) = out;
                continue;
            }
            uint8_t *base = page + (size_t)((is_v ? a.n_kv : 0) + h) * a.kv.head_bytes;
            if (TYPE == kTypeF32) {
                if (some) *reinterpret_cast<v4f *>(base + ((size_t)off * a.dim + e) * 4) = out;
            } else if (TYPE == kTypeF16) {
                typedef _Float16 v4h __attribute__((ext_vector_type(4)));
                if (some) *reinterpret_cast<v4h *>(base + ((size_t)off * a.dim + e) * 2) = __builtin_convertvector(out, v4h);
            } else {
                // (a block is 8 lanes)
                const uint32_t most = max(max(magnitude(y[0]), magnitude(y[1])), max(magnitude(y[2]), magnitude(y[3])));
                const float top = __uint_as_float(row8_max_u32(most)), id = top != 0.0f ? 127.0f / top : 0.0f;
                uint32_t w = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) w |= ((uint32_t)q8_code(y[j], id) & 0xffu) << (8 * j);
                if (some) {
                    *reinterpret_cast<uint32_t *>(base + (size_t)off * a.dim + e) = w;
                    if ((l & 7) == 0)
                        reinterpret_cast<uint16_t *>(base + ((size_t)a.dim << a.kv.page_shift))[off * (a.dim / 32) + e / 32] =
                            (uint16_t)f32_to_f16_rne(top / 127.0f);
                }
            }
        }
    }
}

namespace {

template <int TYPE>
void launch_rows(const RopeArgs &a, int m, hipStream_t st) {
    const dim3 grid((unsigned)(((long long)m * a.waves + 3) / 4));
    if (a.dim == 64) hipLaunchKernelGGL((rope_rows_kernel<TYPE, 16>), grid, dim3(256), 0, st, a);
    else if (a.dim == 256) hipLaunchKernelGGL((rope_rows_kernel<TYPE, 64>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((rope_rows_kernel<TYPE, 32>), grid, dim3(256), 0, st, a);
}

// Whether rope_rows_kernel takes the call; sets the waves of a token.
bool rows_take(RopeArgs &a, int type, int m) {
    if (a.dim != 64 && a.dim != 96 && a.dim != 128 && a.dim != 256) return false;
    const uintptr_t at = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out | (uintptr_t)a.k_out |
                         (uintptr_t)a.qw | (uintptr_t)a.kw;
    if ((at & 15u) != 0 || ((a.ldq | a.ldk | a.ldv) & 3) != 0) return false;
    // (a lane's values rotate together, and their partners are four neighbours too)
    if (a.n_rot % 4 != 0 || (!a.interleaved && a.n_rot % 8 != 0)) return false;
    const int hpw = a.dim == 64 ? 4 : a.dim == 256 ? 1 : 2;
    const int steps = (a.n_heads + hpw - 1) / hpw + (a.n_kv + hpw - 1) / hpw * (type >= 0 ? 2 : 1);
    // About 16384 waves (twice what runs at once) of at least four steps each, and with few tokens about 4096 of as
    // few steps as there are.  Measured: 8192 tokens of 24 steps 77 us with two waves a token, 83 with one; 777 tokens
    // of 24 steps 13 us with six, 18 with 22 (every wave computes its sines).
    const auto least = [](long long x, long long y) { return x < y ? x : y; };
    const long long w = std::max(least((16384 + m - 1) / m, steps / 4), least((4096 + m - 1) / m, steps));
    a.waves = (int)std::max(w, 1LL);
    return (long long)m * a.waves < INT_MAX - 4;
}

bool launch_rope(RopeArgs &a, int type, int m, hipStream_t st, const char *what) {
    if (m <= 0) return true;
    if (rows_take(a, type, m)) {
        if (type == kTypeF32) launch_rows<kTypeF32>(a, m, st);
        else if (type == kTypeF16) launch_rows<kTypeF16>(a, m, st);
        else if (type == kTypeQ8_0) launch_rows<kTypeQ8_0>(a, m, st);
        else launch_rows<-1>(a, m, st);
        return lib_hip(hipGetLastError(), what);
    }
    const long long waves = (long long)m * (a.n_heads + a.n_kv * (type >= 0 ? 2 : 1));
    if (waves <= 0) return true;
    if (waves > INT_MAX) {
        lib_error(-2, "%s: %d tokens are too many", what, m);
        return false;
    }
    const dim3 grid((unsigned)((waves + 3) / 4));
    if (type == kTypeF32) hipLaunchKernelGGL(rope_kernel<kTypeF32>, grid, dim3(256), 0, st, a);
    else if (type == kTypeF16) hipLaunchKernelGGL(rope_kernel<kTypeF16>, grid, dim3(256), 0, st, a);
    else if (type == kTypeQ8_0) hipLaunchKernelGGL(rope_kernel<kTypeQ8_0>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(rope_kernel<-1>, grid, dim3(256), 0, st, a);
    return lib_hip(hipGetLastError(), what);
}

bool rope_fits(const edgexpu_hip_rope *r, int dim, const char *what) {
    if (r == nullptr || r->n_rot <= dim) return true;
    lib_error(-2, "%s: the rotation's %d values exceed the head's %d", what, r->n_rot, dim);
    return false;
}

}  // namespace

}  // namespace exq

using namespace exq;

extern "C" {

edgexpu_hip_rope *edgexpu_hip_rope_create(int n_rot, double base, double scale, const float *factors,
                                          int interleaved) {
    if (n_rot <= 0 || n_rot % 2 != 0 || n_rot > 256 || !(base > 0.0) || !std::isfinite(base) || !std::isfinite(scale)) {
        lib_error(-2, "rope_create: n_rot=%d (even, 2..256), base=%g, scale=%g", n_rot, base, scale);
        return nullptr;
    }
    double turns[128];
    for (int i = 0; i < n_rot / 2; ++i) {
        turns[i] = scale * std::pow(base, -2.0 * i / n_rot) / (factors != nullptr ? (double)factors[i] : 1.0) /
                   6.283185307179586476925;
        if (std::isfinite(turns[i] * INT_MAX)) continue;  // (any position's angle is a number)
        lib_error(-2, "rope_create: pair %d turns by %g a position", i, turns[i]);
        return nullptr;
    }
    if (!lib_ready("rope_create")) return nullptr;
    void *p = nullptr;
    if (!lib_hip(hipMalloc(&p, sizeof(turns)), "rope_create: hipMalloc")) return nullptr;
    edgexpu_hip_rope *r = new (std::nothrow) edgexpu_hip_rope();
    if (r == nullptr || !lib_hip(hipMemcpy(p, turns, sizeof(double) * (n_rot / 2), hipMemcpyHostToDevice), "rope_create")) {
        if (r == nullptr) lib_error(-5, "rope_create: out of host memory");
        (void)hipFree(p);
        delete r;
        return nullptr;
    }
    r->n_rot = n_rot;
    r->interleaved = interleaved != 0;
    r->turns = (double *)p;
    return r;
}

void edgexpu_hip_rope_destroy(edgexpu_hip_rope *r) {
    if (r == nullptr) return;
    (void)hipDeviceSynchronize();
    (void)hipFree(r->turns);
    delete r;
}

int edgexpu_hip_qk_norm_rope_dev(float *q_out, float *k_out, const float *q, long long ldq, const float *k,
                                 long long ldk, int m, int n_heads, int n_kv_heads, int head_dim,
                                 const float *q_weight, const float *k_weight, float eps,
                                 const edgexpu_hip_rope *rope, const int32_t *pos, void *stream) {
    if (m <= 0 || n_heads < 0 || n_kv_heads < 0 || n_heads + (long long)n_kv_heads <= 0 ||
        n_heads + (long long)n_kv_heads > 65535 || head_dim <= 0 || head_dim % 2 != 0 || head_dim > 256 ||
        (n_heads > 0 && (q == nullptr || q_out == nullptr || ldq < (long long)n_heads * head_dim)) ||
        (n_kv_heads > 0 && (k == nullptr || k_out == nullptr || ldk < (long long)n_kv_heads * head_dim)) ||
        (rope != nullptr && pos == nullptr)) {
        lib_error(-2, "qk_norm_rope: null buffer, short rows or bad sizes (m=%d, %d and %d heads of %d)", m, n_heads,
                  n_kv_heads, head_dim);
        return 0;
    }
    if (!rope_fits(rope, head_dim, "qk_norm_rope") || !lib_ready("qk_norm_rope")) return 0;
    RopeArgs a = {};
    a.q = q;
    a.k = k;
    a.ldq = ldq;
    a.ldk = ldk;
    a.q_out = q_out;
    a.k_out = k_out;
    a.qw = q_weight;
    a.kw = k_weight;
    a.eps = eps;
    a.pos = pos;
    a.m = m;
    a.n_heads = n_heads;
    a.n_kv = n_kv_heads;
    a.dim = head_dim;
    if (rope != nullptr) {
        a.turns = rope->turns;
        a.n_rot = rope->n_rot;
        a.interleaved = rope->interleaved;
    }
    return launch_rope(a, -1, m, (hipStream_t)stream, "qk_norm_rope") ? 1 : 0;
}

int edgexpu_hip_kv_append_dev(float *q_out, const float *q, long long ldq, const float *k, long long ldk,
                              const float *v, long long ldv, edgexpu_hip_batch *b, int layer, const float *q_weight,
                              const float *k_weight, float eps, const edgexpu_hip_rope *rope, void *stream) {
    if (!lib_ready("kv_append")) return 0;
    bool capturing = false;
    if (!batch_ready(b, layer, (hipStream_t)stream, "kv_append", &capturing)) return 0;
    const edgexpu_hip_kv *kv = b->kv;
    if (b->plan.tokens.empty()) return 1;
    if (q == nullptr || q_out == nullptr || k == nullptr || v == nullptr || ldq < (long long)b->n_heads * kv->dim ||
        ldk < (long long)kv->n_kv * kv->dim || ldv < (long long)kv->n_kv * kv->dim) {
        lib_error(-2, "kv_append: null buffer or short rows");
        return 0;
    }
    if (!rope_fits(rope, kv->dim, "kv_append")) return 0;
    if (!b->plan.writable) {
        lib_error(-2, "kv_append: a new token's page is held by another sequence too");
        return 0;
    }
    RopeArgs a = {};
    a.q = q;
    a.k = k;
    a.v = v;
    a.ldq = ldq;
    a.ldk = ldk;
    a.ldv = ldv;
    a.q_out = q_out;
    a.qw = q_weight;
    a.kw = k_weight;
    a.eps = eps;
    a.head = b->head();
    a.kv = kv_view(kv, layer);
    a.n_heads = b->n_heads;
    a.n_kv = kv->n_kv;
    a.dim = kv->dim;
    if (rope != nullptr) {
        a.turns = rope->turns;
        a.n_rot = rope->n_rot;
        a.interleaved = rope->interleaved;
    }
    // (a captured call covers any later plan, of fewer tokens; -1: as many as the plan says)
    const int m = (int)b->plan.tokens.size();
    a.m = capturing ? -1 : m;
    if (capturing) {
        batch_recorded(b);
        b->captured_append = true;
    }
    return launch_rope(a, kv->type, m, (hipStream_t)stream, "kv_append") ? 1 : 0;
}

}  // extern "C"
