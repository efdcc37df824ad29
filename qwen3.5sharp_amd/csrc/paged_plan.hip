// Page tables and slots of a batch of requests from their lengths.
//
// Request i holds R_i rows, in the first have_i = ceil(R_i / P) entries of its table, and
// brings T_i tokens, for which it needs need_i = ceil((R_i + T_i) / P) - have_i pages more.
// With c_i the sum of need_j over j < i, o_i that of T_j, and n_free the list's length as the host
// or, in n_listed, the device has it:
//   table[i][have_i + e] = free[c_i + e], e < need_i, if need_i = 0 or c_i + need_i <= n_free, else -1
//   table[i][e] = -1 behind these
//   slots[o_i + t] = P table[i][(R_i + t) / P] + (R_i + t) % P
// One launch: a workgroup forms the two sums of its request from the lengths before it
// (from L2: four loads a thread for a thousand requests) instead of waiting for another one's, and
// writes its share of the entries and slots, which follow from the free list and the kept entries
// alone.  What bounds it is the launch: 64 requests of 250 pages and a token write 64 KB, 3.4
// us; 128 prompts of up to 2048 tokens, 0.8 MB, 3.7.  Past some thousands of requests it is the
// sums, whose loads grow with their square: calls of 1000 requests of a token 5 us, of 10000 38, of
// 65535 1000.
#include "paged_device.h"

namespace q35 {
namespace {

constexpr int PT = 256;

__device__ __forceinline__ long plan_sum(long v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const int lo = __shfl_xor((int)(unsigned)v, o, kWave), hi = __shfl_xor((int)(v >> 32), o, kWave);
        v += ((long)hi << 32) | (unsigned)lo;
    }
    return v;
}

__global__ __launch_bounds__(PT) void paged_plan(int* __restrict__ table, int* lens, const int* rows, const int* tokens,
                                                 const int* __restrict__ free_pages, int n_free,
                                                 const int* __restrict__ n_listed, int64_t* __restrict__ slots,
                                                 size_t n_slots, int* __restrict__ taken, int max_rows, int max_pages,
                                                 int n_pages, int shift) {
    const int tid = threadIdx.x, i = blockIdx.y;
    if (n_listed) n_free = min(max(*n_listed, 0), n_free);
    struct Need {
        int rows, tokens, have, more;
    };
    auto need = [&](int j) {
        Need n;
        n.rows = min(max(rows[j], 0), max_rows);
        n.tokens = min(max(tokens[j], 0), max_rows - n.rows);
        const int up = (1 << shift) - 1;
        n.have = (n.rows + up) >> shift;
        n.more = ((n.rows + n.tokens + up) >> shift) - n.have;
        return n;
    };
    const Need me = need(i);
    long pages = 0, before = 0;                            // c_i, o_i
    for (int j = tid; j < i; j += PT) {
        const Need n = need(j);
        pages += n.more;
        before += n.tokens;
    }
    __shared__ long sums[2][PT / kWave];
    pages = plan_sum(pages);
    before = plan_sum(before);
    if ((tid & 63) == 0) {
        sums[0][tid >> 6] = pages;
        sums[1][tid >> 6] = before;
    }
    __syncthreads();
    pages = before = 0;
#pragma unroll
    for (int w = 0; w < PT / kWave; ++w) {
        pages += sums[0][w];
        before += sums[1][w];
    }
    const bool served = me.more == 0 || pages + me.more <= n_free;
    auto known = [&](int id) { return id >= 0 && id < n_pages ? id : -1; };
    auto taken_page = [&](int e) {                         // of entry e >= have
        return served && e < me.have + me.more ? known(free_pages[pages + e - me.have]) : -1;
    };
    int* const row = table + (size_t)i * max_pages;
    const int at = blockIdx.x * PT + tid, step = gridDim.x * PT;
    for (int e = me.have + at; e < max_pages; e += step) row[e] = taken_page(e);
    for (int t = at; t < me.tokens && (size_t)(before + t) < n_slots; t += step) {
        const int pos = me.rows + t, e = pos >> shift;
        const int page = e < me.have ? known(row[e]) : taken_page(e);
        slots[before + t] = page < 0 ? -1 : ((int64_t)page << shift) + (pos & ((1 << shift) - 1));
    }
    if (at == 0) {
        lens[i] = me.rows;
        taken[i] = served ? me.more : -1;
    }
}

}  // namespace

hipError_t launch_paged_plan(q35m_paged* p, int n, const int* rows, const int* tokens, const int* free_pages, int n_free,
                             const int* n_listed, int64_t* slots, size_t n_slots, int* taken) {
    q35m_ctx* c = p->ctx;
    // Workgroups a request: four a CU over all requests, and none without an entry or a
    // token of its own.
    const int most = (p->map.max_rows() + PT - 1) / PT;
    int x = 4 * c->n_cu / n;
    x = x < 1 ? 1 : x > most ? most : x;
    ProfScope ps(c, K_PAGED_PLAN);
    hipExtLaunchKernelGGL(paged_plan, dim3(x, n), dim3(PT), 0, c->stream, ps.a, ps.b, 0, p->dev_table, p->dev_len, rows, tokens,
                          free_pages, n_free, n_listed, slots, n_slots, taken, p->map.max_rows(), p->map.max_pages(),
                          p->n_pages, p->page_shift);
    return hipGetLastError();
}

}  // namespace q35
