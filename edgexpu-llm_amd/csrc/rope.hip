// Per-head RMSNorm and position rotation of queries and keys in one pass, with
// the key/value cache write (the reference runs them one after the other per
// token and head: RMSNorm of the head, RoPE in its two pairings, a copy into
// the cache window; src/native.c:2536-2544, src/cpu_kernel.c:659-760).
//
//   y = x * (1 / sqrt(mean(x^2) + eps)) * w         squares summed in double
//   (a, b) -> (a cos - b sin, a sin + b cos)        angle = pos * scale * base^(-2i/n_rot) / factor_i
//
// The angle is kept in turns in 64 bits (pos * turns_i) and its whole turns
// are taken off there, so a position of 10^5 has the same accuracy as one of
// 10; what is left is rounded to 32 bits once.
#include <hip/hip_runtime.h>

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
};

// TYPE: the cache's, -1: k goes to k_out.  One wave a head of a token.
template <int TYPE>
__global__ __launch_bounds__(256) void rope_kernel(const RopeArgs a) {
    __shared__ float rows[4][256];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int slots = a.n_heads + a.n_kv * (TYPE >= 0 ? 2 : 1);
    const int m = a.head != nullptr ? reinterpret_cast<const PlanHeader *>(a.head)->n_tokens : a.m;
    const long long id = (long long)blockIdx.x * 4 + wave;
    const int t = (int)(id / slots), s = (int)(id % slots);
    const bool live = t < m;
    const bool is_q = s < a.n_heads, is_v = s >= a.n_heads + a.n_kv;
    const int h = is_q ? s : is_v ? s - a.n_heads - a.n_kv : s - a.n_heads;
    const float *w = is_q ? a.qw : is_v ? nullptr : a.kw;
    float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    int pos = 0, slot = 0;
    if (live) {
        if (a.head != nullptr) {
            const PlanToken *pt = reinterpret_cast<const PlanToken *>(a.head) - (t + 1);
            pos = pt->pos;
            slot = pt->slot;
        } else if (a.pos != nullptr) {
            pos = a.pos[t];
        }
        const float *x = is_q ? a.q + t * a.ldq : is_v ? a.v + t * a.ldv : a.k + t * a.ldk;
        x += (size_t)h * a.dim;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (lane + 64 * j < a.dim) y[j] = x[lane + 64 * j];
    }
    if (w != nullptr) {  // (the same for the whole wave)
        double ss = 0.0;
#pragma unroll
        for (int j = 0; j < 4; ++j) ss += (double)y[j] * (double)y[j];
        const float scale = rms_scale(wave_sum_f64(ss), a.dim, a.eps);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (lane + 64 * j < a.dim) y[j] = y[j] * scale * w[lane + 64 * j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) rows[wave][lane + 64 * j] = y[j];
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
            float sn, cs;
            sincospif(2.0f * (float)turn, &sn, &cs);
            const float o = rows[wave][other];
            y[j] = first ? y[j] * cs - o * sn : o * sn + y[j] * cs;
        }
    }
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
            float top = fabsf(y[j]);
            top = row16_max(top);
            top = fmaxf(top, shfl_xor_f(top, 16));
            if (e >= a.dim) continue;
            // as edgexpu_hip_quantize_q8_0_dev: codes by 127 / max, the scale max / 127 rounded to f16
            const float id = top != 0.0f ? 127.0f / top : 0.0f;
            reinterpret_cast<int8_t *>(base)[(size_t)off * a.dim + e] = (int8_t)(int)rintf(y[j] * id);
            if ((lane & 31) == 0)
                reinterpret_cast<uint16_t *>(base + ((size_t)a.dim << a.kv.page_shift))[off * (a.dim / 32) + e / 32] =
                    (uint16_t)f32_to_f16_rne(top / 127.0f);
        } else if (e < a.dim) {
            if (TYPE == kTypeF16) reinterpret_cast<_Float16 *>(base)[(size_t)off * a.dim + e] = (_Float16)y[j];
            else reinterpret_cast<float *>(base)[(size_t)off * a.dim + e] = y[j];
        }
    }
}

namespace {

bool launch_rope(const RopeArgs &a, int type, int m, hipStream_t st, const char *what) {
    const long long waves = (long long)m * (a.n_heads + a.n_kv * (type >= 0 ? 2 : 1));
    if (waves <= 0) return true;
    if ((waves + 3) / 4 > INT_MAX) {
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
    if (!lib_ready("rope_create")) return nullptr;
    double turns[128];
    for (int i = 0; i < n_rot / 2; ++i)
        turns[i] = scale * std::pow(base, -2.0 * i / n_rot) / (factors != nullptr ? (double)factors[i] : 1.0) /
                   6.283185307179586476925;
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
    // (a captured call covers any later plan of this batch)
    const int m = capturing ? b->max_tokens : (int)b->plan.tokens.size();
    return launch_rope(a, kv->type, m, (hipStream_t)stream, "kv_append") ? 1 : 0;
}

}  // extern "C"
