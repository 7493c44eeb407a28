// Attention of a step's tokens over the paged cache, by the plan of
// attn_plan.h: out = sum_j p_j V_j / sum_j p_j, p_j = exp(scale q.K_j - m).
#include <hip/hip_runtime.h>

#include "kv.h"
#include "lib.h"

namespace exq {

constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
    const float *q;
    float *out;
    const int32_t *head;
    float *part;
    KvView kv;
    float scale;
    int group, page_tokens;
    size_t part_cap;
};

// One value of a cached row.
template <int TYPE>
__device__ __forceinline__ float kv_value(const uint8_t *head, int off, int e, int dim, int page_tokens) {
    if (TYPE == kTypeF32) return reinterpret_cast<const float *>(head)[(size_t)off * dim + e];
    if (TYPE == kTypeF16) return (float)reinterpret_cast<const _Float16 *>(head)[(size_t)off * dim + e];
    const float d = (float)reinterpret_cast<const _Float16 *>(head + (size_t)page_tokens * dim)[off * (dim / 32) + e / 32];
    return (float)reinterpret_cast<const int8_t *>(head)[(size_t)off * dim + e] * d;
}

// One wave a row, its keys one after the other.
template <int TYPE, int DIM>
__global__ __launch_bounds__(256) void attn_kernel(const AttnArgs a) {
    const PlanHeader *hd = reinterpret_cast<const PlanHeader *>(a.head);
    const AttnItem *items = reinterpret_cast<const AttnItem *>(hd + 1);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n_kv = a.kv.n_kv;
    constexpr int E = (DIM + 63) / 64;
    for (long long w = blockIdx.x; w < (long long)hd->n_items * n_kv; w += gridDim.x) {
        const AttnItem it = items[w / n_kv];
        const int h = (int)(w % n_kv);
        for (int r = wave; r < it.n_rows; r += 4) {
            const int row = it.row0 + r, g = row % a.group;
            const PlanToken *pt = reinterpret_cast<const PlanToken *>(a.head) - (row / a.group + 1);
            const int token = pt->order, key1 = it.causal ? min(it.key1, pt->order_pos + 1) : it.key1;
            const size_t at = (((size_t)token * n_kv + h) * a.group + g) * DIM;
            float qv[E], acc[E], m = -INFINITY, l = 0.0f;
#pragma unroll
            for (int j = 0; j < E; ++j) {
                qv[j] = lane + 64 * j < DIM ? a.q[at + lane + 64 * j] : 0.0f;
                acc[j] = 0.0f;
            }
            for (int p = it.key0; p < key1; ++p) {
                const int page = a.head[it.page_at + (p >> a.kv.page_shift)], off = p & (a.page_tokens - 1);
                const uint8_t *k = a.kv.base + (size_t)page * a.kv.page_bytes + (size_t)h * a.kv.head_bytes;
                const uint8_t *v = k + (size_t)n_kv * a.kv.head_bytes;
                float s = 0.0f;
#pragma unroll
                for (int j = 0; j < E; ++j)
                    if (lane + 64 * j < DIM) s = fmaf(qv[j], kv_value<TYPE>(k, off, lane + 64 * j, DIM, a.page_tokens), s);
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) s += shfl_xor_f(s, o);
                s *= a.scale * kLog2e;
                const float mn = fmaxf(m, s);
                const float c = m == -INFINITY ? 0.0f : exp2f(m - mn), e = exp2f(s - mn);
                l = l * c + e;
#pragma unroll
                for (int j = 0; j < E; ++j)
                    if (lane + 64 * j < DIM)
                        acc[j] = fmaf(e, kv_value<TYPE>(v, off, lane + 64 * j, DIM, a.page_tokens), acc[j] * c);
                m = mn;
            }
            if (it.part < 0) {
#pragma unroll
                for (int j = 0; j < E; ++j)
                    if (lane + 64 * j < DIM) a.out[at + lane + 64 * j] = acc[j] / l;
                continue;
            }
            const size_t ps = (size_t)(it.part + r) * n_kv + h;
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (lane + 64 * j < DIM) a.part[ps * DIM + lane + 64 * j] = acc[j];
            if (lane == 0) {
                float *ml = a.part + a.part_cap * DIM + 2 * ps;
                ml[0] = m;
                ml[1] = l;
            }
        }
    }
}

// Rows with several pieces: one wave a row and kv head joins its partial
// results, out = sum_i 2^(m_i - m) acc_i / sum_i 2^(m_i - m) l_i.
template <int DIM>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnArgs a) {
    const PlanHeader *hd = reinterpret_cast<const PlanHeader *>(a.head);
    const int lane = threadIdx.x & 63, n_kv = a.kv.n_kv;
    constexpr int E = (DIM + 63) / 64;
    for (long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); w < (long long)hd->n_joined * n_kv;
         w += 4LL * gridDim.x) {
        const int i = (int)(w / n_kv), h = (int)(w % n_kv);
        const int row = a.head[hd->join_rows + i];
        const int p0 = a.head[hd->join_at + i], p1 = a.head[hd->join_at + i + 1];
        const float *mls = a.part + a.part_cap * DIM;
        float m = -INFINITY, l = 0.0f, acc[E] = {};
        for (int p = p0; p < p1; ++p) m = fmaxf(m, mls[2 * ((size_t)a.head[p] * n_kv + h)]);
        for (int p = p0; p < p1; ++p) {
            const size_t ps = (size_t)a.head[p] * n_kv + h;
            const float mi = mls[2 * ps];
            if (mi == -INFINITY) continue;  // a piece behind the row's last position
            const float c = exp2f(mi - m);
            l += c * mls[2 * ps + 1];
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (lane + 64 * j < DIM) acc[j] = fmaf(c, a.part[ps * DIM + lane + 64 * j], acc[j]);
        }
        const PlanToken *pt = reinterpret_cast<const PlanToken *>(a.head) - (row / a.group + 1);
        float *out = a.out + (((size_t)pt->order * n_kv + h) * a.group + row % a.group) * DIM;
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (lane + 64 * j < DIM) out[lane + 64 * j] = acc[j] / l;
    }
}

namespace {

template <int DIM>
hipError_t launch_attention(const AttnArgs &a, int type, unsigned grid, unsigned join_grid, hipStream_t st) {
    if (type == kTypeF32) hipLaunchKernelGGL((attn_kernel<kTypeF32, DIM>), dim3(grid), dim3(256), 0, st, a);
    else if (type == kTypeF16) hipLaunchKernelGGL((attn_kernel<kTypeF16, DIM>), dim3(grid), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((attn_kernel<kTypeQ8_0, DIM>), dim3(grid), dim3(256), 0, st, a);
    if (join_grid != 0) hipLaunchKernelGGL((attn_join_kernel<DIM>), dim3(join_grid), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace

}  // namespace exq

using namespace exq;

extern "C" int edgexpu_hip_attention_dev(float *out, const float *q, edgexpu_hip_batch *b, int layer, float scale,
                                         void *stream) {
    if (!lib_ready("attention")) return 0;
    bool capturing = false;
    if (!batch_ready(b, layer, (hipStream_t)stream, "attention", &capturing)) return 0;
    if (out == nullptr || q == nullptr || (((uintptr_t)out | (uintptr_t)q) & 15u) != 0) {
        lib_error(-2, "attention: null buffer, or q or out not 16-byte aligned");
        return 0;
    }
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
    a.page_tokens = kv->tables.page_tokens();
    // One workgroup an item and kv head; a captured call, whose plan may be
    // replaced before a replay, takes a fixed grid that walks whatever is there.
    const long long items = (long long)b->plan.items.size() * kv->n_kv;
    const long long joins = ((long long)b->plan.join_rows.size() * kv->n_kv + 3) / 4;
    const unsigned grid = capturing ? 1024u : (unsigned)std::min<long long>(items, 1 << 20);
    const unsigned join_grid = capturing ? 256u : (unsigned)std::min<long long>(joins, 4096);
    if (grid == 0) return 1;
    hipError_t e;
    switch (kv->dim) {
        case 64: e = launch_attention<64>(a, kv->type, grid, join_grid, (hipStream_t)stream); break;
        case 96: e = launch_attention<96>(a, kv->type, grid, join_grid, (hipStream_t)stream); break;
        case 128: e = launch_attention<128>(a, kv->type, grid, join_grid, (hipStream_t)stream); break;
        default: e = launch_attention<256>(a, kv->type, grid, join_grid, (hipStream_t)stream); break;
    }
    return lib_hip(e, "attention") ? 1 : 0;
}
