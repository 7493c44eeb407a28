// The paged key/value cache: its handle, the copies that its bookkeeping asks
// for, and the step's batch (attention's plan on the device).
//
// The reference keeps one sequence's f32 window [layer][pos][kv_head][head_dim]
// (src/kv_cache.c:22-127).  Here many sequences share one pool of pages:
// bookkeeping on the host (kv_tables.h), and the only device work is copying
// the pages it names.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstring>
#include <new>
#include <utility>

#include "kv.h"
#include "lib.h"

namespace exq {

// A piece of attention of less than 8 us costs more in its start and its
// partial results than it gains.  Measured with 5, 8, 12 and 24 us: 4 tokens
// each of 2 sequences behind 12499 f32 keys 17, 18, 18 and 25 us; 20 each of 8
// behind 3000 Q8_0 keys 44, 34, 34 and 38; one f16 sequence of 700 11, 12, 13, 13.
constexpr int kMinPieceCost = 80000;

// Copies of pages, at most kMovesMax a launch, given as kernel arguments (no
// transfer of a list in front of the kernel).
constexpr int kMovesMax = 256;
struct MoveArgs {
    int src[kMovesMax], dst[kMovesMax];
    uint16_t used[kMovesMax];
};

// One workgroup copies one (move, layer, K or V and head): `used` rows of
// row_bytes, and behind the page's rows `used` rows of scale_bytes (Q8_0).
// Bytes are read once and written once; nothing is computed.  Bound by them:
// 10.8 GB in 2.0 ms (24 sequences of up to 1500 tokens, 32 layers of 8 heads of
// 128 in f16: half the pool moved, half copied), 5.4 TB/s; 32 last pages of 36
// tokens on average 67 us, 4.6 TB/s.
__global__ __launch_bounds__(256) void kv_copy_kernel(uint8_t *__restrict__ pool, size_t layer_bytes, size_t page_bytes,
                                                      unsigned head_bytes, unsigned row_bytes, unsigned scale_bytes,
                                                      int page_tokens, const MoveArgs mv) {
    const int m = blockIdx.x;
    const size_t at = (size_t)blockIdx.z * layer_bytes + (size_t)blockIdx.y * head_bytes;
    const uint8_t *src = pool + at + (size_t)mv.src[m] * page_bytes;
    uint8_t *dst = pool + at + (size_t)mv.dst[m] * page_bytes;
    const unsigned used = mv.used[m];
    const unsigned n = used * row_bytes;  // a multiple of 16
    for (unsigned i = threadIdx.x * 16; i < n; i += 256 * 16)
        *reinterpret_cast<uint4 *>(dst + i) = *reinterpret_cast<const uint4 *>(src + i);
    if (scale_bytes == 0) return;
    const unsigned s0 = (unsigned)page_tokens * row_bytes, ns = used * scale_bytes;  // a multiple of 2
    for (unsigned i = threadIdx.x * 2; i < ns; i += 256 * 2)
        *reinterpret_cast<uint16_t *>(dst + s0 + i) = *reinterpret_cast<const uint16_t *>(src + s0 + i);
}

namespace {

size_t head_page_bytes(uint32_t type, int head_dim, int page_tokens) {
    const size_t n = (size_t)head_dim * page_tokens;
    return type == (uint32_t)kTypeF32 ? n * 4 : type == (uint32_t)kTypeF16 ? n * 2 : n + n / 16;
}

bool kv_shape_ok(uint32_t type, int n_layers, int n_kv, int dim, int page, int n_pages) {
    if (type != (uint32_t)kTypeF32 && type != (uint32_t)kTypeF16 && type != (uint32_t)kTypeQ8_0) return false;
    if (dim != 64 && dim != 96 && dim != 128 && dim != 256) return false;
    if (page != 16 && page != 32 && page != 64 && page != 128 && page != 256) return false;
    // (grid limits of the copy kernel: 2 * n_kv and n_layers below 65536)
    if (n_layers <= 0 || n_layers > 4096 || n_kv <= 0 || n_kv > 4096 || n_pages <= 0 || (long long)n_pages * page >= INT_MAX)
        return false;
    return (double)n_layers * n_pages * 2 * n_kv * (double)head_page_bytes(type, dim, page) < 0x1p60;
}

const char *status_text(KvStatus s) {
    switch (s) {
        case KvStatus::bad_seq: return "a sequence number that is not in use";
        case KvStatus::repeated: return "the same sequence twice";
        case KvStatus::bad_count: return "a token count out of range";
        case KvStatus::no_pages: return "the pool has not enough free pages";
        case KvStatus::no_seqs: return "every sequence number is in use";
        default: return "ok";
    }
}

bool status_ok(KvStatus s, const char *what) {
    if (s == KvStatus::ok) return true;
    lib_error(s == KvStatus::no_pages || s == KvStatus::no_seqs ? -6 : -2, "%s: %s", what, status_text(s));
    return false;
}

bool is_capturing(hipStream_t st) {
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(st, &cs) != hipSuccess) {  // the null stream beside a capture
        (void)hipGetLastError();
        return true;
    }
    return cs != hipStreamCaptureStatusNone;
}

bool refuse_capture(hipStream_t st, const char *what) {
    if (!is_capturing(st)) return false;
    lib_error(-7, "%s: not while a stream is captured", what);
    return true;
}

bool run_moves(edgexpu_hip_kv *kv, hipStream_t st, const char *what) {
    const unsigned row = kv->type == kTypeF32 ? kv->dim * 4u : kv->type == kTypeF16 ? kv->dim * 2u : (unsigned)kv->dim;
    const unsigned scale = kv->type == kTypeQ8_0 ? (unsigned)kv->dim / 16 : 0u;
    for (size_t i = 0; i < kv->moves.size(); i += kMovesMax) {
        const int n = (int)std::min<size_t>(kMovesMax, kv->moves.size() - i);
        MoveArgs mv;
        for (int j = 0; j < n; ++j) {
            mv.src[j] = kv->moves[i + j].src;
            mv.dst[j] = kv->moves[i + j].dst;
            mv.used[j] = (uint16_t)kv->moves[i + j].used;
        }
        hipLaunchKernelGGL(kv_copy_kernel, dim3(n, 2 * kv->n_kv, kv->n_layers), dim3(256), 0, st, kv->pool,
                           kv->layer_bytes(), kv->page_bytes(), (unsigned)kv->head_bytes, row, scale,
                           kv->tables.page_tokens(), mv);
        if (!lib_hip(hipGetLastError(), what)) return false;
    }
    return true;
}

// Host code below may run out of memory inside std::vector; nothing thrown passes a C entry.
template <typename F, typename R>
R guarded(const char *what, R fail, F f) {
    try {
        return f();
    } catch (...) {
        lib_error(-5, "%s: out of host memory", what);
        return fail;
    }
}

}  // namespace

bool batch_ready(edgexpu_hip_batch *b, int layer, hipStream_t st, const char *what, bool *capturing) {
    if (b == nullptr || layer < 0 || layer >= b->kv->n_layers) {
        lib_error(-2, "%s: null batch or layer %d out of range", what, layer);
        return false;
    }
    if (!b->set || b->epoch != b->kv->tables.epoch()) {
        lib_error(-2, "%s: the batch is %s", what, b->set ? "stale: the cache's sequences have changed since it was set"
                                                         : "not set");
        return false;
    }
    *capturing = is_capturing(st);
    return true;
}

void batch_recorded(edgexpu_hip_batch *b) {
    b->captured = true;
    b->captured_tokens = std::min(b->captured_tokens, (int)b->plan.tokens.size());
}

}  // namespace exq

using namespace exq;

extern "C" {

size_t edgexpu_hip_kv_pool_bytes(uint32_t type, int n_layers, int n_kv_heads, int head_dim, int page_tokens,
                                 int n_pages) {
    if (!kv_shape_ok(type, n_layers, n_kv_heads, head_dim, page_tokens, n_pages)) return 0;
    return (size_t)n_layers * n_pages * 2 * n_kv_heads * head_page_bytes(type, head_dim, page_tokens);
}

edgexpu_hip_kv *edgexpu_hip_kv_create(void *dev_pool, uint32_t type, int n_layers, int n_kv_heads, int head_dim,
                                      int page_tokens, int n_pages, int max_seqs) {
    if (!kv_shape_ok(type, n_layers, n_kv_heads, head_dim, page_tokens, n_pages) || max_seqs <= 0 ||
        ((uintptr_t)dev_pool & 15u) != 0) {
        lib_error(-2,
                  "kv_create: type %u, %d layers, %d kv heads of %d, %d pages of %d tokens, %d sequences: not a "
                  "supported shape, or the pool is not 16-byte aligned",
                  type, n_layers, n_kv_heads, head_dim, n_pages, page_tokens, max_seqs);
        return nullptr;
    }
    if (!lib_ready("kv_create")) return nullptr;
    edgexpu_hip_kv *kv = guarded("kv_create", (edgexpu_hip_kv *)nullptr,
                                 [&] { return new edgexpu_hip_kv(page_tokens, n_pages, max_seqs); });
    if (kv == nullptr) return nullptr;
    kv->type = (int)type;
    kv->n_layers = n_layers;
    kv->n_kv = n_kv_heads;
    kv->dim = head_dim;
    kv->head_bytes = head_page_bytes(type, head_dim, page_tokens);
    kv->pool = (uint8_t *)dev_pool;
    if (dev_pool == nullptr) {
        void *p = nullptr;
        if (!lib_hip(hipMalloc(&p, (size_t)n_layers * kv->layer_bytes()), "kv_create: hipMalloc")) {
            delete kv;
            return nullptr;
        }
        kv->pool = (uint8_t *)p;
        kv->owned = true;
    }
    return kv;
}

int edgexpu_hip_kv_destroy(edgexpu_hip_kv *kv) {
    if (kv == nullptr) return 1;
    if (kv->n_batches > 0) {
        lib_error(-2, "kv_destroy: %d batches of this cache live", kv->n_batches);
        return 0;
    }
    if (kv->owned) {
        (void)hipDeviceSynchronize();
        (void)hipFree(kv->pool);
    }
    delete kv;
    return 1;
}

void *edgexpu_hip_kv_pool(const edgexpu_hip_kv *kv) { return kv == nullptr ? nullptr : kv->pool; }
int edgexpu_hip_kv_free_pages(const edgexpu_hip_kv *kv) { return kv == nullptr ? 0 : kv->tables.free_pages(); }

int edgexpu_hip_kv_new(edgexpu_hip_kv *kv) {
    if (kv == nullptr) {
        lib_error(-2, "kv_new: null cache");
        return -1;
    }
    const int s = kv->tables.new_seq();
    if (s < 0) lib_error(-6, "kv_new: every sequence number is in use");
    return s;
}

int edgexpu_hip_kv_fork(edgexpu_hip_kv *kv, int n, const int *parents, int copy, int *children, void *stream) {
    if (kv == nullptr || n < 0 || (n > 0 && (parents == nullptr || children == nullptr))) {
        lib_error(-2, "kv_fork: null argument or n=%d", n);
        return 0;
    }
    if (copy && (!lib_ready("kv_fork") || refuse_capture((hipStream_t)stream, "kv_fork"))) return 0;
    return guarded("kv_fork", 0, [&] {
        kv->moves.clear();
        if (!status_ok(kv->tables.fork(n, parents, copy != 0, children, kv->moves), "kv_fork")) return 0;
        return run_moves(kv, (hipStream_t)stream, "kv_fork") ? 1 : 0;
    });
}

int edgexpu_hip_kv_extend(edgexpu_hip_kv *kv, int n, const int *seqs, const int *n_new, void *stream) {
    if (kv == nullptr || n < 0 || (n > 0 && (seqs == nullptr || n_new == nullptr))) {
        lib_error(-2, "kv_extend: null argument or n=%d", n);
        return 0;
    }
    if (!lib_ready("kv_extend") || refuse_capture((hipStream_t)stream, "kv_extend")) return 0;
    return guarded("kv_extend", 0, [&] {
        kv->moves.clear();
        if (!status_ok(kv->tables.extend(n, seqs, n_new, kv->moves), "kv_extend")) return 0;
        return run_moves(kv, (hipStream_t)stream, "kv_extend") ? 1 : 0;
    });
}

int edgexpu_hip_kv_truncate(edgexpu_hip_kv *kv, int seq, int n_tokens) {
    if (kv == nullptr) {
        lib_error(-2, "kv_truncate: null cache");
        return 0;
    }
    return status_ok(kv->tables.truncate(seq, n_tokens), "kv_truncate") ? 1 : 0;
}

int edgexpu_hip_kv_release(edgexpu_hip_kv *kv, int n, const int *seqs) {
    if (kv == nullptr || n < 0 || (n > 0 && seqs == nullptr)) {
        lib_error(-2, "kv_release: null argument or n=%d", n);
        return 0;
    }
    return status_ok(kv->tables.release(n, seqs), "kv_release") ? 1 : 0;
}

int edgexpu_hip_kv_compact(edgexpu_hip_kv *kv, int *n_used, void *stream) {
    if (kv == nullptr) {
        lib_error(-2, "kv_compact: null cache");
        return 0;
    }
    if (!lib_ready("kv_compact") || refuse_capture((hipStream_t)stream, "kv_compact")) return 0;
    return guarded("kv_compact", 0, [&] {
        kv->moves.clear();
        const int used = kv->tables.compact(kv->moves);
        if (n_used != nullptr) *n_used = used;
        return run_moves(kv, (hipStream_t)stream, "kv_compact") ? 1 : 0;
    });
}

int edgexpu_hip_kv_length(const edgexpu_hip_kv *kv, int seq) {
    return kv != nullptr && kv->tables.valid(seq) ? kv->tables.seq(seq).len : -1;
}

int edgexpu_hip_kv_tables(const edgexpu_hip_kv *kv, int n, const int *seqs, int *out, int ld) {
    if (kv == nullptr || n < 0 || (n > 0 && seqs == nullptr)) {
        lib_error(-2, "kv_tables: null argument or n=%d", n);
        return -1;
    }
    int most = 0;
    for (int i = 0; i < n; ++i) {
        if (!kv->tables.valid(seqs[i])) {
            lib_error(-2, "kv_tables: a sequence number that is not in use");
            return -1;
        }
        most = std::max(most, (int)kv->tables.seq(seqs[i]).pages.size());
    }
    if (out == nullptr) return most;
    if (ld < most) {
        lib_error(-2, "kv_tables: ld=%d below %d pages", ld, most);
        return -1;
    }
    for (int i = 0; i < n; ++i) {
        const std::vector<int> &p = kv->tables.seq(seqs[i]).pages;
        int *row = out + (size_t)i * ld;
        for (int j = 0; j < ld; ++j) row[j] = j < (int)p.size() ? p[j] : -1;
    }
    return most;
}

// ------------------------------------------------------------------ the step's batch

edgexpu_hip_batch *edgexpu_hip_batch_create(edgexpu_hip_kv *kv, int n_heads, int max_seqs, int max_tokens) {
    if (kv == nullptr || n_heads <= 0 || n_heads % kv->n_kv != 0 || n_heads > 65535 || max_seqs <= 0 ||
        max_tokens <= 0 || (long long)max_tokens * n_heads >= INT_MAX / 4) {
        lib_error(-2, "batch_create: null cache, %d heads not a multiple of its kv heads, or bad sizes (%d, %d)", n_heads,
                  max_seqs, max_tokens);
        return nullptr;
    }
    if (!lib_ready("batch_create") || !lib_hip(attn_prepare(kv->type, kv->dim), "batch_create")) return nullptr;
    edgexpu_hip_batch *b =
        guarded("batch_create", (edgexpu_hip_batch *)nullptr, [] { return new edgexpu_hip_batch(); });
    if (b == nullptr) return nullptr;
    b->kv = kv;
    b->n_heads = n_heads;
    b->max_seqs = max_seqs;
    b->max_tokens = max_tokens;
    kv->n_batches++;
    return b;
}

void edgexpu_hip_batch_destroy(edgexpu_hip_batch *b) {
    if (b == nullptr) return;
    (void)hipDeviceSynchronize();
    if (b->words) (void)hipFree(b->words);
    if (b->part) (void)hipFree(b->part);
    for (int i = 0; i < edgexpu_hip_batch::kStages; ++i) {
        if (b->stage[i]) (void)hipHostFree(b->stage[i]);
        if (b->done[i]) (void)hipEventDestroy(b->done[i]);
    }
    b->kv->n_batches--;
    delete b;
}

int edgexpu_hip_batch_tokens(const edgexpu_hip_batch *b) {
    return b != nullptr && b->set ? (int)b->plan.tokens.size() : 0;
}

namespace {

// Device memory of at least front + n * each bytes in *p, with room for half as
// much again; *cap becomes the count that fits.  Refused, with nothing changed,
// while a captured call holds the pointer.  What it held goes: the batch is not set.
bool grow(edgexpu_hip_batch *b, void **p, size_t front, size_t n, size_t each, size_t *cap, const char *what) {
    if (n <= *cap) return true;
    if (b->captured) {
        lib_error(-7, "batch_set: the plan outgrows the %s that a captured call uses (set the largest plan before it)",
                  what);
        return false;
    }
    b->set = false;
    if (!lib_hip(hipDeviceSynchronize(), "batch_set: sync")) return false;
    if (*p) (void)hipFree(*p);
    *p = nullptr;
    *cap = 0;
    const size_t bytes = (front + (n + n / 2) * each + 65535) / 65536 * 65536;
    if (!lib_hip(hipMalloc(p, bytes), "batch_set: hipMalloc")) return false;
    *cap = (bytes - front) / each;
    return true;
}

bool upload(edgexpu_hip_batch *b, hipStream_t st) {
    const AttnPlan &pl = b->made;
    const size_t T = pl.tokens.size(), items_at = sizeof(PlanHeader) / 4, pages_at = items_at + 8 * pl.items.size(),
                 rows_at = pages_at + pl.pages.size(), joins_at = rows_at + pl.join_rows.size(),
                 parts_at = joins_at + pl.join_at.size(), words = parts_at + pl.join_parts.size();
    if (!grow(b, (void **)&b->words, 16 * (size_t)b->max_tokens, words, 4, &b->words_cap, "plan buffer")) return false;
    // a partial result: dim values, its maximum and its sum
    if (!grow(b, (void **)&b->part, 0, (size_t)pl.parts * b->kv->n_kv, ((size_t)b->kv->dim + 2) * 4, &b->part_cap,
              "workspace"))
        return false;
    const int k = b->next;
    b->next = (k + 1) % edgexpu_hip_batch::kStages;
    if (b->busy[k] && !lib_hip(hipEventSynchronize(b->done[k]), "batch_set: event")) return false;
    b->busy[k] = false;
    const size_t n = 4 * T + words;
    if (n > b->stage_cap[k]) {
        if (b->stage[k]) (void)hipHostFree(b->stage[k]);
        b->stage[k] = nullptr;
        b->stage_cap[k] = 0;
        const size_t cap = n + n / 2 + 4096;
        if (!lib_hip(hipHostMalloc((void **)&b->stage[k], cap * 4, hipHostMallocDefault), "batch_set: hipHostMalloc"))
            return false;
        b->stage_cap[k] = cap;
    }
    if (b->done[k] == nullptr &&
        !lib_hip(hipEventCreateWithFlags(&b->done[k], hipEventDisableTiming), "batch_set: event"))
        return false;
    int32_t *h = b->stage[k] + 4 * T;
    for (size_t t = 0; t < T; ++t) memcpy(h - 4 * (t + 1), &pl.tokens[t], 16);
    PlanHeader hd = {};
    hd.n_tokens = (int)T;
    hd.n_items = (int)pl.items.size();
    hd.n_joined = (int)pl.join_rows.size();
    hd.join_rows = (int)rows_at;
    hd.join_at = (int)joins_at;
    hd.parts = pl.parts;
    memcpy(h, &hd, sizeof(hd));
    for (size_t i = 0; i < pl.items.size(); ++i) {
        AttnItem it = pl.items[i];
        it.page_at += (int)pages_at;
        memcpy(h + items_at + 8 * i, &it, 32);
    }
    const auto put = [&](size_t at, const std::vector<int32_t> &v) {
        if (!v.empty()) memcpy(h + at, v.data(), v.size() * 4);
    };
    put(pages_at, pl.pages);
    put(rows_at, pl.join_rows);
    for (size_t i = 0; i < pl.join_at.size(); ++i) h[joins_at + i] = pl.join_at[i] + (int)parts_at;
    put(parts_at, pl.join_parts);
    b->set = false;
    if (!lib_hip(hipMemcpyAsync(b->head() - 4 * T, b->stage[k], n * 4, hipMemcpyHostToDevice, st), "batch_set: copy"))
        return false;
    b->busy[k] = true;
    return lib_hip(hipEventRecord(b->done[k], st), "batch_set: event");
}

}  // namespace

int edgexpu_hip_batch_set(edgexpu_hip_batch *b, int n, const int *seqs, const int *n_new, void *stream) {
    if (b == nullptr || n < 0 || n > b->max_seqs || (n > 0 && (seqs == nullptr || n_new == nullptr))) {
        lib_error(-2, "batch_set: null argument, or %d sequences (at most %d)", n, b == nullptr ? 0 : b->max_seqs);
        return 0;
    }
    if (!lib_ready("batch_set") || refuse_capture((hipStream_t)stream, "batch_set")) return 0;
    KvTables &kt = b->kv->tables;
    if (!status_ok(kt.distinct(n, seqs), "batch_set")) return 0;
    long long tokens = 0;
    for (int i = 0; i < n; ++i) {
        if (n_new[i] < 0 || n_new[i] > kt.seq(seqs[i]).len) {
            lib_error(-2, "batch_set: %d new tokens of a sequence of %d", n_new[i], kt.seq(seqs[i]).len);
            return 0;
        }
        tokens += n_new[i];
    }
    if (tokens > b->max_tokens) {
        lib_error(-2, "batch_set: %lld tokens (at most %d)", tokens, b->max_tokens);
        return 0;
    }
    if (tokens > b->captured_tokens) {
        lib_error(-7, "batch_set: a plan of %lld tokens outgrows a captured call made for %d (set the largest plan before it)",
                  tokens, b->captured_tokens);
        return 0;
    }
    return guarded("batch_set", 0, [&] {
        const edgexpu_hip_kv *kv = b->kv;
        // (a partial result: its bytes twice, at a workgroup's part of 5.1 TB/s)
        const int at_once = attn_workgroups(kv->type, kv->dim);
        b->made.build(kt, n, seqs, n_new,
                      {b->n_heads / kv->n_kv, kv->n_kv, attn_cost(kv->type, kv->dim), (kv->dim + 2) * 4 * 2 * at_once / 512,
                       at_once, kMinPieceCost});
        if (b->captured_append && !b->made.writable) {
            lib_error(-2, "batch_set: a captured call appends, and a new token's page is held by another sequence too");
            return 0;
        }
        if (!upload(b, (hipStream_t)stream)) return 0;
        std::swap(b->plan, b->made);
        b->epoch = kt.epoch();
        b->set = true;
        return 1;
    });
}

}  // extern "C"
