// The products of a step's tokens with the experts they were routed to.
//
//   act[t][j] = f(b_g[e] + W_g[e] . q8(x[t])) * (b_u[e] + W_u[e] . q8(x[t]))
//   out[t]    = [residual[t] +] sum_j w[t][j] (b[e] + W[e] . q8(act[t][j]))
//   e = ids[t][j]
#include <algorithm>
#include <cmath>
#include <new>

#include "formats.h"
#include "lib.h"
#include "moe.h"

hipError_t launch_quantize_q8_0(const float *x, int m, int K, int ldx, uint8_t *packed, hipStream_t st);
hipError_t launch_quantize_q8_k(const float *x, int m, int K, int ldx, uint8_t *packed, hipStream_t st);

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
    const uint8_t *w[2];      // gate and up, or down
    const float *bias[2];
    const uint8_t *xq;        // quantized rows
    size_t xq_stride, row_bytes;
    size_t expert_bytes;
    float *out;
    const float *residual;
    int m, top_k, rows, nblk, activation;
};

// What a format's load_w and load_act read.
struct MoeRow {
    const uint8_t *w;
    size_t row_bytes;
    const uint8_t *xq;
    size_t xq_stride;
};

template <class F>
__device__ float moe_dot(const MoeRow &r, int row, int token, int units, int lane) {
    float acc = 0.0f;
    for (int u = lane; u < units; u += 64) {
        typename F::Act x;
        typename F::W w;
        F::load_act(r, u, token, x);
        F::load_w(r, row, u, w);
        F::dot1(w, u, x, acc);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) acc += shfl_xor_f(acc, off);
    return acc;
}

// A wave a row of gate and up.
template <class F>
__global__ __launch_bounds__(256) void moe_gate_up_kernel(MoeArgs a) {
    const int lane = threadIdx.x & 63;
    const int row = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);
    if (row >= a.rows) return;
    for (size_t pair = blockIdx.y; pair < (size_t)a.m * a.top_k; pair += gridDim.y) {
        const int e = a.ids[pair];
        float v = 0.0f;
        if (e >= 0) {
            float y[2];
            for (int z = 0; z < 2; ++z) {
                const MoeRow r = {a.w[z] + (size_t)e * a.expert_bytes, a.row_bytes, a.xq, a.xq_stride};
                y[z] = moe_dot<F>(r, row, (int)(pair / a.top_k), a.nblk * F::kUnitsPerBlock, lane);
                if (a.bias[z] != nullptr) y[z] = a.bias[z][(size_t)e * a.rows + row] + y[z];
            }
            v = moe_act(y[0], a.activation) * y[1];
        }
        if (lane == 0) a.out[pair * a.rows + row] = v;
    }
}

// A wave a row of a token's experts.
template <class F>
__global__ __launch_bounds__(256) void moe_down_kernel(MoeArgs a) {
    const int lane = threadIdx.x & 63;
    const int row = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);
    if (row >= a.rows) return;
    for (int t = (int)blockIdx.y; t < a.m; t += (int)gridDim.y) {
        float s = 0.0f;
        for (int j = 0; j < a.top_k; ++j) {
            const size_t pair = (size_t)t * a.top_k + j;
            const int e = a.ids[pair];
            if (e < 0) continue;
            const MoeRow r = {a.w[0] + (size_t)e * a.expert_bytes, a.row_bytes, a.xq, a.xq_stride};
            float y = moe_dot<F>(r, row, (int)pair, a.nblk * F::kUnitsPerBlock, lane);
            if (a.bias[0] != nullptr) y = a.bias[0][(size_t)e * a.rows + row] + y;
            s = fmaf(a.weights[pair], y, s);
        }
        if (lane == 0) {
            const size_t at = (size_t)t * a.rows + row;
            a.out[at] = a.residual != nullptr ? a.residual[at] + s : s;
        }
    }
}

namespace {

template <class F>
void moe_launch(const MoeArgs &a, bool pair, hipStream_t st) {
    const long long n = pair ? (long long)a.m * a.top_k : a.m;
    const dim3 grid((unsigned)((a.rows + 3) / 4), (unsigned)(n < 65535 ? n : 65535));
    if (pair)
        hipLaunchKernelGGL(moe_gate_up_kernel<F>, grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL(moe_down_kernel<F>, grid, dim3(256), 0, st, a);
}

bool moe_product(MoeArgs &a, uint32_t type, bool pair, const float *x, long long m, int K, hipStream_t st,
                 const char *what) {
    if (!lib_hip(k_family((int)type) ? launch_quantize_q8_k(x, (int)m, K, K, (uint8_t *)a.xq, st)
                                     : launch_quantize_q8_0(x, (int)m, K, K, (uint8_t *)a.xq, st), what))
        return false;
    switch ((int)type) {
        case kTypeQ4_0: moe_launch<FmtQ40>(a, pair, st); break;
        case kTypeQ5_0: moe_launch<FmtQ50>(a, pair, st); break;
        case kTypeQ8_0: moe_launch<FmtQ80>(a, pair, st); break;
        case kTypeQ4_K: moe_launch<FmtQ4K>(a, pair, st); break;
        case kTypeQ5_K: moe_launch<FmtQ5K>(a, pair, st); break;
        default: moe_launch<FmtQ6K>(a, pair, st); break;
    }
    return lib_hip(hipGetLastError(), what);
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

// Bytes of n quantized elements in either activation format.
size_t q8_bytes(int n) { return ((size_t)n + 31) / 32 * kBytesQ8_0 + ((size_t)n + 255) / 256 * (kBytesQ8_K - 272); }

MoeArgs moe_args(const edgexpu_hip_moe *p, uint32_t type, int rows, int K) {
    MoeArgs a = {};
    a.ids = p->ids;
    a.weights = p->weights;
    a.nblk = K / (k_family((int)type) ? kQKK : kQK8_0);
    a.row_bytes = a.nblk * block_bytes(type);
    a.expert_bytes = a.row_bytes * (size_t)rows;
    a.xq = p->xq;
    a.xq_stride = (size_t)a.nblk * (k_family((int)type) ? kBytesQ8_K : kBytesQ8_0);
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
    const size_t xq = std::max(q8_bytes(n_embd) * max_tokens, q8_bytes(n_ff) * pairs);
    const size_t total = 2 * up(4 * pairs) + up(xq);
    if (!lib_hip(hipMalloc((void **)&p->mem, total), "moe_create: hipMalloc")) {
        delete p;
        return nullptr;
    }
    p->ids = (int32_t *)p->mem;
    p->weights = (float *)(p->mem + up(4 * pairs));
    p->xq = p->mem + 2 * up(4 * pairs);
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
    p->m = m;
    return 1;
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
    p->m = m;
    return 1;
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
    a.out = act;
    return moe_product(a, type, true, x, p->m, p->n_embd, (hipStream_t)stream, what) ? 1 : 0;
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
    a.out = out;
    return moe_product(a, type, false, act, (long long)p->pairs(), p->n_ff, (hipStream_t)stream, what) ? 1 : 0;
}

}  // extern "C"
