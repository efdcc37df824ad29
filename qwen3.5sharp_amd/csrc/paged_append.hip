// Paged K/V cache: the rows of new tokens put into their pages, and the small
// kernels that keep the device copies of page tables and lengths.
//
// K row = norm(rope(k, p)) (1 + w) at the token's position p, V row = v, both
// rounded once to the cache's type: the cache write of DecodeAttention /
// PrefillAttention (src/Qwen35Sharp.Model/Qwen35Model.Decode.cs:294-311,
// Ops.cs:75-160, Qwen35Ops.cs:22-66).
#include "paged_device.h"

namespace q35 {
namespace {

constexpr int kTableIds = 900;       // page ids of one update, in its kernel arguments

struct TableSet {
    int n;
    int id[kTableIds];
};

__global__ __launch_bounds__(256) void paged_table_set(int* __restrict__ table, TableSet s) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t < s.n) table[t] = s.id[t];
}

struct LengthSet {
    int n;
    int seq[kMaxBatch];
    int len[kMaxBatch];
};

__global__ __launch_bounds__(64) void paged_lengths_set(int* __restrict__ lens, LengthSet s) {
    const int t = threadIdx.x;
    if (t < s.n) lens[s.seq[t]] = s.len[t];
}

struct Freqs {
    float f[kRopeHalf];
};

// Ops.EnsureRopeTable (src/Qwen35Sharp.Model/Ops.cs:135-160): the angle is the
// fp32 product of position and frequency, as there; its cosine and sine are
// kept in 64 bits (see paged_key_row).
__global__ __launch_bounds__(256) void paged_rope_fill(double* __restrict__ table, int rows, Freqs f) {
    const size_t t = (size_t)blockIdx.x * 256 + threadIdx.x;
    const size_t row = t / kRopeHalf;
    const int i = (int)(t % kRopeHalf);
    if (row >= (size_t)rows) return;
    const double angle = (double)__fmul_rn((float)(int)row, f.f[i]);
    table[row * kRopeDim + i] = cos(angle);
    table[row * kRopeDim + kRopeHalf + i] = sin(angle);
}

// One wave per (new row, kv head), four a workgroup, from unit0 on.  Reads 2 KiB and
// writes 2 rows a wave: a copy with a reduction of one wave in between.  In 4 bits a lane
// rounds its own four values with its block's power of two, the largest of 8 lanes; 2048 rows of 4
// kv heads, 19 MB, 7.2 us, of which a launch and a chain of loads (arguments, table, row) are 2.5.
template <typename T, int N>
__global__ __launch_bounds__(256) void paged_append_rows(PagedView pv, PagedBatchOf<N> b, const float* __restrict__ k,
                                                         const float* __restrict__ v, const float* __restrict__ k_norm,
                                                         double eps, long unit0) {
    const int lane = threadIdx.x & 63;
    const long unit = unit0 + (long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = (int)(unit / pv.nkv), kvh = (int)(unit % pv.nkv);
    if (row >= b.off[b.n]) return;
    const size_t at = ((size_t)row * pv.nkv + kvh) * kHd + 4 * lane;
    const float4 xk = *reinterpret_cast<const float4*>(k + at);
    const float4 xv = *reinterpret_cast<const float4*>(v + at);
    // The row's sequence: the last one that starts at or before it.
    const int i = __popcll(__ballot(lane < b.n && b.off[min(lane, b.n)] <= row)) - 1;
    const int seq = b.seq[i];
    const int pos = pv.lens[seq] + row - b.off[i];
    if (pos >= pv.max_rows) return;
    const int page = page_of(pv.table + (size_t)seq * pv.max_pages, pos >> pv.page_shift, pv.max_pages, pv.n_pages);
    if (page < 0) return;
    const float4 y = paged_key_row<std::is_same_v<T, Mx4>>(xk, pv.rope + (size_t)pos * kRopeDim, k_norm, lane, eps);
    if constexpr (std::is_same_v<T, Mx4>) {
        const int in = pos & ((1 << pv.page_shift) - 1);
        mx_put_key((uint8_t*)pv.k + mx_page(pv, page, kvh), pv, in, mx_round(y), lane);
        mx_put_value((uint8_t*)pv.v + mx_page(pv, page, kvh), pv, in, mx_round(xv), lane);
    } else {
        const size_t to = row_offset<T>(pv, page, kvh, pos) + 4 * lane;
        store_row4((T*)pv.k + to, y);
        store_row4((T*)pv.v + to, xv);
    }
}

// Rows read back, one wave per (row, kv head): row `row` of the call is row first + (its
// place) of its sequence.  Rows of pages that are not mapped are zeros.
// Bound by what it writes: 2048 rows of 4 kv heads in 4 bits, 2.2 MB read and 16.8 written, 6.7 us.
template <typename T, int N>
__global__ __launch_bounds__(256) void paged_rows(PagedView pv, PagedBatchOf<N> b, PagedFirstOf<N> first,
                                                  float* __restrict__ k, float* __restrict__ v, long unit0) {
    const int lane = threadIdx.x & 63;
    const long unit = unit0 + (long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = (int)(unit / pv.nkv), kvh = (int)(unit % pv.nkv);
    if (row >= b.off[b.n]) return;
    const int i = __popcll(__ballot(lane < b.n && b.off[min(lane, b.n)] <= row)) - 1;
    const int pos = first.row[i] + row - b.off[i];
    const int page = page_of(pv.table + (size_t)b.seq[i] * pv.max_pages, pos >> pv.page_shift, pv.max_pages, pv.n_pages);
    float4 xk = make_float4(0.f, 0.f, 0.f, 0.f), xv = xk;
    if (page >= 0) {
        if constexpr (std::is_same_v<T, Mx4>) {
            const int in = pos & ((1 << pv.page_shift) - 1);
            const uint8_t* const kp = (const uint8_t*)pv.k + mx_page(pv, page, kvh);
            const uint8_t* const vp = (const uint8_t*)pv.v + mx_page(pv, page, kvh);
            const uint32_t at = (uint32_t)in * kMxCodes + 2 * lane;
            xk = mx_values({*reinterpret_cast<const uint16_t*>(kp + at), kp[mx_key_scale(pv, in) + (lane >> 3)]});
            xv = mx_values({*reinterpret_cast<const uint16_t*>(vp + at), vp[mx_value_scale(pv, in, lane >> 3)]});
        } else {
            const size_t at = row_offset<T>(pv, page, kvh, pos) + 4 * lane;
            xk = load_row4((const T*)pv.k + at);
            xv = load_row4((const T*)pv.v + at);
        }
    }
    const size_t to = ((size_t)row * pv.nkv + kvh) * kHd + 4 * lane;
    *reinterpret_cast<float4*>(k + to) = xk;
    *reinterpret_cast<float4*>(v + to) = xv;
}

}  // namespace

hipError_t launch_paged_rope(q35m_ctx* c, double* table, int rows) {
    Freqs f;
    for (int i = 0; i < kRopeHalf; ++i) f.f[i] = 1.0f / powf(c->d.rope_base, (float)i / (float)kRopeHalf);
    const size_t n = (size_t)rows * kRopeHalf;
    hipLaunchKernelGGL(paged_rope_fill, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, c->stream, table, rows, f);
    return hipGetLastError();
}

hipError_t launch_paged_table(q35m_ctx* c, int* table, size_t at, const int* ids, int n) {
    for (int done = 0; done < n; done += kTableIds) {
        TableSet s;
        s.n = n - done < kTableIds ? n - done : kTableIds;
        for (int i = 0; i < s.n; ++i) s.id[i] = ids ? ids[done + i] : -1;
        hipLaunchKernelGGL(paged_table_set, dim3((s.n + 255) / 256), dim3(256), 0, c->stream, table + at + done, s);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_paged_lengths(q35m_ctx* c, int* lens, int n, const int* seq, const int* len) {
    LengthSet s;
    s.n = n;
    for (int i = 0; i < n; ++i) {
        s.seq[i] = seq[i];
        s.len[i] = len[i];
    }
    hipLaunchKernelGGL(paged_lengths_set, dim3(1), dim3(64), 0, c->stream, lens, s);
    return hipGetLastError();
}

hipError_t launch_paged_append(q35m_paged* p, int layer, const PagedBatch& b, const float* k, const float* v) {
    q35m_ctx* c = p->ctx;
    // (a grid holds fewer than 2^32 threads, 2^26 units)
    constexpr long kMost = 1L << 22;
    const long units = (long)b.off[b.n] * c->d.nkv;
    return with_batch(b, [&](const auto& some) {
        constexpr int N = std::decay_t<decltype(some)>::kSeqs;
        for (long u = 0; u < units; u += kMost) {
            ProfScope ps(c, K_PAGED_APPEND);
            auto go = [&](auto kern) {
                const long n = units - u < kMost ? units - u : kMost;
                hipExtLaunchKernelGGL(kern, dim3((unsigned)((n + 3) / 4)), dim3(256), 0, c->stream, ps.a, ps.b, 0,
                                      p->view(layer), some, k, v, c->full[layer].k_norm, (double)c->d.eps, u);
            };
            if (p->type == Q35M_KV_MXFP4) go(paged_append_rows<Mx4, N>);
            else if (p->type == Q35M_KV_F16) go(paged_append_rows<_Float16, N>);
            else go(paged_append_rows<float, N>);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        return hipSuccess;
    });
}

hipError_t launch_paged_rows(q35m_paged* p, int layer, const PagedBatch& b, const PagedFirst& first, float* k, float* v) {
    q35m_ctx* c = p->ctx;
    constexpr long kMost = 1L << 22;
    const long units = (long)b.off[b.n] * c->d.nkv;
    return with_batch(b, [&](const auto& some) {
        constexpr int N = std::decay_t<decltype(some)>::kSeqs;
        PagedFirstOf<N> from;
        for (int i = 0; i < N; ++i) from.row[i] = i < b.n ? first.row[i] : 0;
        for (long u = 0; u < units; u += kMost) {
            ProfScope ps(c, K_PAGED_ROWS);
            auto go = [&](auto kern) {
                const long n = units - u < kMost ? units - u : kMost;
                hipExtLaunchKernelGGL(kern, dim3((unsigned)((n + 3) / 4)), dim3(256), 0, c->stream, ps.a, ps.b, 0,
                                      p->view(layer), some, from, k, v, u);
            };
            if (p->type == Q35M_KV_MXFP4) go(paged_rows<Mx4, N>);
            else if (p->type == Q35M_KV_F16) go(paged_rows<_Float16, N>);
            else go(paged_rows<float, N>);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        return hipSuccess;
    });
}

}  // namespace q35
