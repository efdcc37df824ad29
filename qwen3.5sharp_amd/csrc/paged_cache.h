// Internal declarations of the paged K/V cache: the handle, the batch of a
// call and the launchers (paged_cache.cpp holds the C entry points).
#pragma once

#include <vector>

#include "page_map.h"
#include "q35mix_internal.h"

namespace q35 {

// Sequences of one call and, per sequence, its first row in the call's
// activations (off[n]: all rows), by value in the kernel arguments.  Lengths
// and page tables are read from device memory, so a captured launch stays
// valid as they change.
struct PagedBatch {
    int n;
    int seq[kMaxBatch];
    int off[kMaxBatch + 1];
};

// What the kernels know of one layer's pages.  A page holds page_rows rows of
// every kv head, head-major: [page][kv_head][row][head_dim].
struct PagedView {
    void* k;
    void* v;
    const int* table;       // [n_seqs][max_pages], -1: not mapped
    const int* lens;        // [n_seqs]
    const double* rope;     // [max_rows][64]: 32 cosines, 32 sines
    int max_pages, n_pages;
    int page_shift;         // log2 of page_rows
    int max_rows;
    int nkv;
};

constexpr int kPagedDecodeHeads = 16;    // q heads a decode workgroup takes at most
constexpr int kPagedTileRows = 64;       // query rows of a prefill workgroup

}  // namespace q35

struct q35m_paged {
    q35m_ctx* ctx = nullptr;
    q35::PageMap map;
    int type = 0;                        // Q35M_KV_F32, Q35M_KV_F16
    int n_pages = 0, page_shift = 0;
    std::vector<void*> k, v;             // by layer (null for DeltaNet layers)
    size_t layer_bytes = 0;              // of K, and of V, of one layer
    int* dev_table = nullptr;
    int* dev_len = nullptr;
    double* rope = nullptr;
    float* work = nullptr;               // partial results of one attention call
    size_t work_bytes = 0;
    std::vector<void*> allocations;

    q35m_paged(int n_seqs, int max_rows, int n_pages_, int page_rows)
        : map(n_seqs, max_rows, n_pages_, page_rows), n_pages(n_pages_) {}
    // Whether the stream is being captured: a replay's lengths are not known now.
    bool capturing() const {
        hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
        return hipStreamIsCapturing(ctx->stream, &st) != hipSuccess || st != hipStreamCaptureStatusNone;
    }
    size_t value_bytes() const { return type == Q35M_KV_F16 ? 2 : 4; }
    q35::PagedView view(int layer) const {
        return {k[layer], v[layer], dev_table, dev_len, rope, map.max_pages(), n_pages, page_shift,
                map.max_rows(), ctx->d.nkv};
    }
};

namespace q35 {

// The rotation's table, [rows][32 cosines, 32 sines].
hipError_t launch_paged_rope(q35m_ctx* c, double* table, int rows);
// table[at .. at + n) = ids (null: -1).
hipError_t launch_paged_table(q35m_ctx* c, int* table, size_t at, const int* ids, int n);
// lens[seq[i]] = len[i] for i < n (n at most kMaxBatch).
hipError_t launch_paged_lengths(q35m_ctx* c, int* lens, int n, const int* seq, const int* len);

hipError_t launch_paged_append(q35m_paged* p, int layer, const PagedBatch& b, const float* k, const float* v);
size_t paged_decode_work_bytes(const q35m_ctx* c);
hipError_t launch_paged_decode(q35m_paged* p, int layer, const PagedBatch& b, const float* q_gate, const float* k,
                               const float* v, float* out);
size_t paged_prefill_work_bytes(const q35m_ctx* c);
hipError_t launch_paged_prefill(q35m_paged* p, int layer, const PagedBatch& b, const float* q_gate, float* out);

}  // namespace q35
