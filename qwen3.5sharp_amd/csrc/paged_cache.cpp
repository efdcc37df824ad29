// Paged K/V cache: lifecycle, argument checks and C entry points of the
// paged part of include/q35mix.h.  Page tables and lengths have a host copy
// (page_map.h), which every call is checked against, and a device copy, which
// the kernels read; a change of the host copy enqueues the same change of the
// device copy on the context's stream, so calls enqueued before it see the old
// state and calls after it the new one.
#include <algorithm>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <initializer_list>
#include <new>

#include "paged_cache.h"

int q35_set_error(int code, const char* msg);

namespace {

int pfail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int pfail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return q35_set_error(code, buf);
}

// (HIP keeps an error for the thread's next hipGetLastError, which is that of a later
// launch: it is taken back once it is reported.)
int phip(hipError_t e, const char* what) {
    (void)hipGetLastError();
    return pfail(e == hipErrorOutOfMemory ? Q35M_ERR_OOM : Q35M_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

#define PHIP_TRY(expr, what)                          \
    do {                                              \
        const hipError_t e_ = (expr);                 \
        if (e_ != hipSuccess) return phip(e_, what);  \
    } while (0)

// The context's device made current for a call, and the caller's put back.  An error
// that an earlier call of the thread left is not this call's: a launch that succeeded
// would be reported as failed, and its change of lengths or pages not be kept.
class DeviceScope {
public:
    explicit DeviceScope(int device) {
        (void)hipGetLastError();
        if (hipGetDevice(&before_) != hipSuccess) before_ = device;
        if (before_ != device) (void)hipSetDevice(device);
        else before_ = -1;
    }
    ~DeviceScope() {
        if (before_ >= 0) (void)hipSetDevice(before_);
    }

private:
    int before_ = -1;
};

int map_fail(const q35m_paged* p, q35::PageMap::Result r, int seq) {
    using M = q35::PageMap;
    switch (r) {
        case M::kOk: return Q35M_OK;
        case M::kBadSeq: return pfail(Q35M_ERR_INVALID, "sequence %d out of range [0, %d)", seq, p->map.n_seqs());
        case M::kBadRange:
            return pfail(Q35M_ERR_RANGE, "sequence %d has page entries [0, %d)", seq, p->map.max_pages());
        case M::kBadPage: return pfail(Q35M_ERR_INVALID, "page ids are in [0, %d)", p->n_pages);
        case M::kShared:
            return pfail(Q35M_ERR_INVALID, "sequence %d: a page of the new rows is mapped by another entry too "
                         "(shared pages are read-only)", seq);
        case M::kUnmapped:
            return pfail(Q35M_ERR_CAPACITY, "sequence %d: the pages of its rows up to the new ones are not all mapped",
                         seq);
        case M::kTooLong:
            return pfail(Q35M_ERR_CAPACITY, "sequence %d: the new rows exceed the %d rows of a sequence", seq,
                         p->map.max_rows());
    }
    return pfail(Q35M_ERR_INVALID, "sequence %d", seq);
}

int check_layer(const q35m_paged* p, int layer, bool weights) {
    const q35m_ctx* c = p->ctx;
    if (layer < 0 || layer >= c->cfg.num_layers)
        return pfail(Q35M_ERR_INVALID, "layer %d out of range [0, %d)", layer, c->cfg.num_layers);
    if (c->is_recurrent[layer]) return pfail(Q35M_ERR_INVALID, "layer %d is a Gated-DeltaNet layer", layer);
    if (weights && !c->full[layer].has_weights) return pfail(Q35M_ERR_INVALID, "layer %d has no weights", layer);
    return Q35M_OK;
}

int check_pointers(std::initializer_list<const void*> ptrs) {
    for (const void* x : ptrs) {
        if (!x) return pfail(Q35M_ERR_INVALID, "null activation pointer");
        if ((uintptr_t)x & 15) return pfail(Q35M_ERR_INVALID, "activation pointers must be 16-byte aligned");
    }
    return Q35M_OK;
}

// Distinct sequences of the cache, at most kMaxBatch.
int check_seqs(const q35m_paged* p, int n, const int* seqs) {
    if (n < 1 || n > q35::kMaxBatch)
        return pfail(Q35M_ERR_CAPACITY, "batch of %d sequences (1..%d per call)", n, q35::kMaxBatch);
    if (!seqs) return pfail(Q35M_ERR_INVALID, "null seqs");
    for (int i = 0; i < n; ++i) {
        if (!p->map.has(seqs[i])) return map_fail(p, q35::PageMap::kBadSeq, seqs[i]);
        for (int j = 0; j < i; ++j)
            if (seqs[j] == seqs[i]) return pfail(Q35M_ERR_INVALID, "sequence %d repeated", seqs[i]);
    }
    return Q35M_OK;
}

// The batch of a call that writes tokens[i] rows (null: one) of each sequence, up to
// `most` in all.
int build_batch(const q35m_paged* p, int n, const int* seqs, const int* tokens, bool need_tokens, long most,
                q35::PagedBatch* b) {
    int r = check_seqs(p, n, seqs);
    if (r) return r;
    if (need_tokens && !tokens) return pfail(Q35M_ERR_INVALID, "null tokens");
    long sum = 0;
    b->n = n;
    b->off[0] = 0;
    for (int i = 0; i < n; ++i) {
        const int t = need_tokens ? tokens[i] : 1;
        if (t < 0) return pfail(Q35M_ERR_INVALID, "sequence %d: %d tokens", seqs[i], t);
        sum += t;
        if (sum > most) return pfail(Q35M_ERR_UNSUPPORTED, "more than %ld new rows in one call", most);
        b->seq[i] = seqs[i];
        b->off[i + 1] = (int)sum;
    }
    for (int i = 0; i < n; ++i) {
        const q35::PageMap::Result m = p->map.usable(seqs[i], b->off[i + 1] - b->off[i]);
        if (m != q35::PageMap::kOk) return map_fail(p, m, seqs[i]);
    }
    return Q35M_OK;
}

// New rows of one call: an append, and a prefill, whose query rows (of all heads) are
// what the grids count: of more than 2^27, q_gate and out would not fit the device.
constexpr long kMostRows = 1L << 24, kMostQueryRows = 1L << 27;
constexpr int kMostHeads = 4096;    // a tile's rows are within 2^31 bytes of its first

int not_capturing(const q35m_paged* p, const char* what) {
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    PHIP_TRY(hipStreamIsCapturing(p->ctx->stream, &st), what);
    if (st != hipStreamCaptureStatusNone)
        return pfail(Q35M_ERR_INVALID, "%s: the stream is being captured (a replay would repeat the change)", what);
    return Q35M_OK;
}

void release(q35m_paged* p) {
    if (p->ctx->stream) (void)hipStreamSynchronize(p->ctx->stream);
    for (void* x : p->allocations) (void)hipFree(x);
    p->allocations.clear();
}

int alloc(q35m_paged* p, void** x, size_t bytes, bool zero) {
    *x = nullptr;
    PHIP_TRY(hipMalloc(x, bytes), "hipMalloc");
    p->allocations.push_back(*x);
    if (zero) PHIP_TRY(hipMemsetAsync(*x, 0, bytes, p->ctx->stream), "hipMemsetAsync");
    return Q35M_OK;
}

int fill(q35m_paged* p, int page_rows) {
    q35m_ctx* c = p->ctx;
    const int layers = c->cfg.num_layers;
    p->k.assign(layers, nullptr);
    p->v.assign(layers, nullptr);
    p->allocations.reserve(2 * (size_t)layers + 4);
    p->layer_bytes = (size_t)p->n_pages * c->d.nkv * page_rows * q35::kHd * p->value_bytes();
    const size_t entries = (size_t)p->map.n_seqs() * p->map.max_pages();
    int r = Q35M_OK;
    for (int l = 0; l < layers && !r; ++l) {
        if (c->is_recurrent[l]) continue;
        r = alloc(p, &p->k[l], p->layer_bytes, true);
        if (!r) r = alloc(p, &p->v[l], p->layer_bytes, true);
    }
    if (!r) r = alloc(p, (void**)&p->dev_table, entries * sizeof(int), false);
    if (!r) r = alloc(p, (void**)&p->dev_len, (size_t)p->map.n_seqs() * sizeof(int), true);
    if (!r) r = alloc(p, (void**)&p->rope, (size_t)p->map.max_rows() * q35::kRopeDim * sizeof(double), false);
    const size_t wd = q35::paged_decode_work_bytes(c), wp = q35::paged_prefill_work_bytes(c);
    p->work_bytes = wd > wp ? wd : wp;
    if (!r) r = alloc(p, (void**)&p->work, p->work_bytes, false);
    if (r) return r;
    PHIP_TRY(hipMemsetAsync(p->dev_table, 0xff, entries * sizeof(int), c->stream), "hipMemsetAsync");
    PHIP_TRY(q35::launch_paged_rope(c, p->rope, p->map.max_rows()), "rotation table");
    PHIP_TRY(hipStreamSynchronize(c->stream), "paged cache");
    return Q35M_OK;
}

}  // namespace

extern "C" {

int q35m_paged_create(q35m_ctx* ctx, int n_seqs, int max_rows, int n_pages, int page_rows, int kv_type,
                      q35m_paged** out) {
    if (!out) return pfail(Q35M_ERR_INVALID, "null output pointer");
    *out = nullptr;
    if (!ctx) return pfail(Q35M_ERR_INVALID, "null context");
    if (n_seqs < 1 || max_rows < 1 || n_pages < 1)
        return pfail(Q35M_ERR_INVALID, "n_seqs, max_rows and n_pages must be positive");
    if (max_rows > (1 << 24)) return pfail(Q35M_ERR_UNSUPPORTED, "max_rows %d: up to 2^24", max_rows);
    if ((long)max_rows * ctx->d.nh > (1L << 30))     // the kernels count units of 64 rows and head groups in 32 bits
        return pfail(Q35M_ERR_UNSUPPORTED, "max_rows %d: up to 2^30 over the %d q heads", max_rows, ctx->d.nh);
    if (ctx->d.nh > kMostHeads) return pfail(Q35M_ERR_UNSUPPORTED, "%d q heads: up to %d", ctx->d.nh, kMostHeads);
    int shift = 4;
    while (shift <= 10 && (1 << shift) != page_rows) ++shift;
    if (shift > 10) return pfail(Q35M_ERR_UNSUPPORTED, "page_rows %d: a power of two from 16 to 1024", page_rows);
    if (kv_type != Q35M_KV_F32 && kv_type != Q35M_KV_F16) return pfail(Q35M_ERR_INVALID, "unknown cache type %d", kv_type);
    bool any = false;
    for (int l = 0; l < ctx->cfg.num_layers; ++l) any |= ctx->is_recurrent[l] == 0;
    if (!any) return pfail(Q35M_ERR_INVALID, "the context has no full-attention layer");
    DeviceScope dev(ctx->device);
    q35m_paged* p = nullptr;
    int r;
    try {
        p = new q35m_paged(n_seqs, max_rows, n_pages, page_rows);
        p->ctx = ctx;
        p->type = kv_type;
        p->page_shift = shift;
        r = not_capturing(p, "paged_create");
        if (!r) r = fill(p, page_rows);
    } catch (const std::bad_alloc&) {
        r = pfail(Q35M_ERR_OOM, "paged_create: out of host memory");
    }
    if (r) {
        if (p) release(p);
        delete p;
        return r;
    }
    *out = p;
    return Q35M_OK;
}

int q35m_paged_destroy(q35m_paged* p) {
    if (!p) return Q35M_OK;
    DeviceScope dev(p->ctx->device);
    release(p);
    delete p;
    return Q35M_OK;
}

int q35m_paged_map(q35m_paged* p, int seq, int first, int n, const int* pages) {
    if (!p) return pfail(Q35M_ERR_INVALID, "null paged cache");
    DeviceScope dev(p->ctx->device);
    int r = not_capturing(p, "paged_map");
    if (r) return r;
    const q35::PageMap::Result m = p->map.can_map(seq, first, n, pages);
    if (m != q35::PageMap::kOk) return map_fail(p, m, seq);
    PHIP_TRY(q35::launch_paged_table(p->ctx, p->dev_table, (size_t)seq * p->map.max_pages() + first, pages, n),
             "paged_map");
    (void)p->map.map(seq, first, n, pages);
    return Q35M_OK;
}

int q35m_paged_advance(q35m_paged* p, int n, const int* seqs, const int* tokens) {
    if (!p) return pfail(Q35M_ERR_INVALID, "null paged cache");
    DeviceScope dev(p->ctx->device);
    int r = check_seqs(p, n, seqs);
    if (r) return r;
    if (!tokens) return pfail(Q35M_ERR_INVALID, "null tokens");
    if ((r = not_capturing(p, "paged_advance"))) return r;
    int len[q35::kMaxBatch];
    for (int i = 0; i < n; ++i) {
        if (tokens[i] < 0) return pfail(Q35M_ERR_INVALID, "negative advance %d", tokens[i]);
        if ((long)p->map.length(seqs[i]) + tokens[i] > p->map.max_rows())
            return map_fail(p, q35::PageMap::kTooLong, seqs[i]);
        len[i] = p->map.length(seqs[i]) + tokens[i];
    }
    PHIP_TRY(q35::launch_paged_lengths(p->ctx, p->dev_len, n, seqs, len), "paged_advance");
    for (int i = 0; i < n; ++i) p->map.set_length(seqs[i], len[i]);
    return Q35M_OK;
}

int q35m_paged_truncate(q35m_paged* p, int seq, int length) {
    if (!p) return pfail(Q35M_ERR_INVALID, "null paged cache");
    DeviceScope dev(p->ctx->device);
    if (!p->map.has(seq)) return map_fail(p, q35::PageMap::kBadSeq, seq);
    if (length < 0) return pfail(Q35M_ERR_INVALID, "negative length %d", length);
    if (length > p->map.length(seq))
        return pfail(Q35M_ERR_RANGE, "cannot extend sequence %d from %d to %d", seq, p->map.length(seq), length);
    int r = not_capturing(p, "paged_truncate");
    if (r) return r;
    PHIP_TRY(q35::launch_paged_lengths(p->ctx, p->dev_len, 1, &seq, &length), "paged_truncate");
    p->map.set_length(seq, length);
    return Q35M_OK;
}

int q35m_paged_len(const q35m_paged* p, int seq, int* length) {
    if (!p) return pfail(Q35M_ERR_INVALID, "null paged cache");
    if (!p->map.has(seq)) return map_fail(p, q35::PageMap::kBadSeq, seq);
    if (!length) return pfail(Q35M_ERR_INVALID, "null length");
    *length = p->map.length(seq);
    return Q35M_OK;
}

int q35m_paged_device_ptr(q35m_paged* p, int layer, int kind, void** dptr, size_t* bytes) {
    if (!p) return pfail(Q35M_ERR_INVALID, "null paged cache");
    int r = check_layer(p, layer, false);
    if (r) return r;
    if (kind != Q35M_STATE_KEYS && kind != Q35M_STATE_VALUES)
        return pfail(Q35M_ERR_INVALID, "a paged cache holds keys and values (kind %d)", kind);
    if (dptr) *dptr = kind == Q35M_STATE_KEYS ? p->k[layer] : p->v[layer];
    if (bytes) *bytes = p->layer_bytes;
    return Q35M_OK;
}

int q35m_paged_append(q35m_paged* p, int layer, int n, const int* seqs, const int* tokens, const float* k,
                      const float* v) {
    if (!p) return pfail(Q35M_ERR_INVALID, "null paged cache");
    int r = check_layer(p, layer, true);
    q35::PagedBatch b;
    if (!r) r = build_batch(p, n, seqs, tokens, true, kMostRows, &b);
    if (!r) r = check_pointers({k, v});
    if (r || b.off[n] == 0) return r;
    DeviceScope dev(p->ctx->device);
    PHIP_TRY(q35::launch_paged_append(p, layer, b, k, v), "paged_append");
    return Q35M_OK;
}

int q35m_paged_attn_decode(q35m_paged* p, int layer, int n, const int* seqs, const float* q_gate, const float* k,
                           const float* v, float* out) {
    if (!p) return pfail(Q35M_ERR_INVALID, "null paged cache");
    int r = check_layer(p, layer, true);
    q35::PagedBatch b;
    if (!r) r = build_batch(p, n, seqs, nullptr, false, kMostRows, &b);
    if (!r) r = check_pointers({q_gate, k, v, out});
    if (r) return r;
    DeviceScope dev(p->ctx->device);
    PHIP_TRY(q35::launch_paged_decode(p, layer, b, q_gate, k, v, out), "paged_attn_decode");
    return Q35M_OK;
}

int q35m_paged_attn_prefill(q35m_paged* p, int layer, int n, const int* seqs, const int* tokens,
                            const float* q_gate, const float* k, const float* v, float* out) {
    if (!p) return pfail(Q35M_ERR_INVALID, "null paged cache");
    int r = check_layer(p, layer, true);
    q35::PagedBatch b;
    if (!r) r = build_batch(p, n, seqs, tokens, true, std::min(kMostRows, kMostQueryRows / p->ctx->d.nh), &b);
    if (!r) r = check_pointers({q_gate, k, v, out});
    if (r || b.off[n] == 0) return r;
    DeviceScope dev(p->ctx->device);
    PHIP_TRY(q35::launch_paged_append(p, layer, b, k, v), "paged_attn_prefill rows");
    PHIP_TRY(q35::launch_paged_prefill(p, layer, b, q_gate, out), "paged_attn_prefill");
    return Q35M_OK;
}

}  // extern "C"
