// Paged K/V cache: attention of chunks of new tokens, several sequences a call.
//
// Row j of a sequence's chunk sits at position p = length + j and attends over
// the sequence's rows 0 .. p (its chunk's rows among them, which
// paged_append_rows has put into their pages): s = q . K / 16, softmax, P V,
// times sigmoid(gate): PrefillAttention after the projections
// (src/Qwen35Sharp.Model/Qwen35Model.Prefill.cs:113-149).
//
// A query tile is 64 query rows: 64 / hg tokens of the hg q heads that share a
// kv head, so each K and V row brought in serves 64 rows.  Work is counted in
// units of one query tile by 64 cache rows and dealt out evenly: workgroup w
// takes units [w per, (w + 1) per) of all tiles of all sequences in order.  The
// query tiles of a sequence are ordered first, last, second, last but one, ...:
// under the causal mask such a pair has the same number of units wherever it
// lies, so a prompt of two tiles a workgroup has no tile cut.  A stretch of
// units of one query tile (a segment) that is the whole tile is finished where
// it is; of the others (a workgroup's first and last at most) maximum, sum and
// unnormalised output go to the workspace for paged_prefill_merge.  Lengths
// are read on the device, so a captured launch fits any.
//
// The products are the bound (4 x 256 flop a q head and visible row).
// Scores are formed as S^T = K Q^T and the output as O^T = V^T P^T: P^T's operand
// is S^T's own register layout, so P never crosses lanes, and the softmax's
// statistics of a query row are one lane's (and its partner's) registers.
#include "paged_device.h"

namespace q35 {
namespace {

constexpr int NT = 256;
constexpr int kUnit = 64;               // cache rows of a unit
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPShift = 7.0f;         // P = e^{s - m} 2^7: see paged_decode.hip
constexpr float kLazy = 8.0f;           // log2 of how far a score may pass the running maximum before it moves

// ---- the units of a call ------------------------------------------------

// Query tiles of one (sequence, head group) and their units.  Tile j (TM = 64 /
// hg tokens) has cnt(j) = ceil((start + (j + 1) TM) / 64) units (the last tile,
// if short, may count one more than it has rows for), which is
// floor((q0 + j) / hg); sums of such floors are closed forms.
struct Tiles {
    int shift;             // log2 hg
    int n;                 // tiles
    long q0;
    __device__ __forceinline__ Tiles(int start, int tokens, int hg_shift) : shift(hg_shift) {
        const int tm_shift = 6 - hg_shift, tm = 1 << tm_shift;
        n = (tokens + tm - 1) >> tm_shift;
        q0 = ((long)start + tm + kUnit - 1) >> tm_shift;
    }
    __device__ __forceinline__ long floors(long m) const {      // sum of floor(y / hg) over y < m
        const long k = m >> shift;
        return ((k * (k - 1)) >> 1 << shift) + k * (m - (k << shift));
    }
    __device__ __forceinline__ long cnt(int j) const { return (q0 + j) >> shift; }
    __device__ __forceinline__ long before(int j) const { return floors(q0 + j) - floors(q0); }   // tiles < j
    // In the paired order: the tile at place o, and the units of the places before o.
    __device__ __forceinline__ int tile(int o) const { return o & 1 ? n - 1 - (o >> 1) : o >> 1; }
    __device__ __forceinline__ long ordered(int o) const {
        const int p = o >> 1;
        return before(p) + before(n) - before(n - p) + (o & 1 ? cnt(p) : 0);
    }
};

__device__ __forceinline__ long shfl_up_long(long v, int o) {
    const int lo = __shfl_up((int)(unsigned)v, o, kWave), hi = __shfl_up((int)(v >> 32), o, kWave);
    return ((long)hi << 32) | (unsigned)lo;
}
__device__ __forceinline__ long readlane_long(long v, int i) {
    const int lo = __builtin_amdgcn_readlane((int)(unsigned)v, i), hi = __builtin_amdgcn_readlane((int)(v >> 32), i);
    return ((long)hi << 32) | (unsigned)lo;
}

// A value that is the same in every lane, as one the compiler knows to be.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ long uniform(long v) {
    return ((long)uniform((int)(v >> 32)) << 32) | (unsigned)uniform((int)(unsigned)v);
}

// Lane i: the units of the call's sequences up to and with the i-th.
struct Units {
    int start;
    long end, total;
};
__device__ __forceinline__ Units units_of(const PagedView& pv, const PagedBatch& b, int groups, int hg_shift, int lane) {
    Units u;
    u.start = 0;
    u.end = 0;
    if (lane < b.n) {
        u.start = pv.lens[b.seq[lane]];
        const Tiles t(u.start, b.off[lane + 1] - b.off[lane], hg_shift);
        u.end = t.before(t.n) * groups;
    }
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const long x = shfl_up_long(u.end, o);
        if (lane >= o) u.end += x;
    }
    u.total = readlane_long(u.end, kWave - 1);
    return u;
}

// A workgroup's walk over its units, segment by segment.
struct Walk {
    long u, u_end;
    // the current segment: sequence i of the batch, head group y, query tile j, units [t0, t1) of `tiles`
    int i, y, j, t0, t1, tiles, start, tokens;
    int o, n;

    __device__ __forceinline__ void begin(const Units& un, int wg, int nwg) {
        const long per = uniform((un.total + nwg - 1) / nwg);
        u = wg * per;
        u_end = min(u + per, un.total);
        i = -1;
    }
    // The segment at u; false past the end.
    __device__ __forceinline__ bool next(const PagedBatch& b, const Units& un, int groups, int hg_shift) {
        if (u >= u_end) return false;
        long within;
        if (i >= 0 && t1 == tiles && o + 1 < n) {        // the next tile of the same head group
            ++o;
            within = 0;
        } else {
            i = uniform((int)__popcll(__ballot(un.end <= u)));
            start = __builtin_amdgcn_readlane(un.start, i);
            tokens = b.off[i + 1] - b.off[i];
            const Tiles ts(start, tokens, hg_shift);
            n = ts.n;
            const long each = ts.before(n);
            long rest = u - (readlane_long(un.end, i) - each * groups);
            y = (int)(rest / each);
            rest -= (long)y * each;
            int lo = 0, hi = n - 1;                      // last place whose units begin at or before rest
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (ts.ordered(mid) <= rest) lo = mid;
                else hi = mid - 1;
            }
            o = lo;
            within = rest - ts.ordered(o);
        }
        const Tiles ts(start, tokens, hg_shift);
        y = uniform(y);
        o = uniform(o);
        n = uniform(n);
        j = ts.tile(o);
        tiles = uniform((int)ts.cnt(j));
        t0 = uniform((int)within);
        t1 = uniform((int)min((long)tiles, within + (u_end - u)));
        u = uniform(u + t1 - t0);
        return true;
    }
};

// ---- fp16 cache -----------------------------------------------------------

// 16 bytes a lane from global memory straight to LDS at address at + 16 lane (at
// the same in every lane).  Complete once vmcnt says so: dma_wait() before the
// barrier that publishes the rows.  The instruction is written out because the
// compiler, told of it, waits for all such loads before the next LDS read, also
// one of the other buffer.
__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(const lds_void*)p; }
__device__ __forceinline__ void dma16(const void* p, uint32_t at) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(p) : "memory");
}
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// V rows of a unit that not every query row of the tile sees.  Rows past the
// tile's last row hold anything and become zeros; a value that is not finite
// becomes zero too (0 x inf is NaN in the products of the query rows that do not
// see it), and the outputs of the query rows that do are marked in `poison`, a
// bit a (query row, dim), which turns them to NaN at the segment's end.  A wave
// takes `count` rows of kHd values from v on; base: their first row's position.
__device__ __forceinline__ bool not_finite(float x) { return !(fabsf(x) < INFINITY); }
__device__ __forceinline__ bool not_finite(_Float16 x) {
    return (__builtin_bit_cast(unsigned short, x) & 0x7c00) == 0x7c00;
}
template <typename T>
__device__ __forceinline__ void guard_rows(T* v, int count, int base, int rows, uint32_t (*poison)[kHd / 32], int first,
                                           int tokens_left, int hg_shift, int lane) {
    constexpr int E = 16 / sizeof(T);          // values of 16 bytes
    typedef T vec __attribute__((ext_vector_type(E)));
#pragma nounroll
    for (int x = lane; x < count * (kHd / E); x += kWave) {
        const int r = base + x / (kHd / E);
        vec y = *reinterpret_cast<vec*>(v + x * E);
        bool bad = false;
#pragma unroll
        for (int k = 0; k < E; ++k) bad |= not_finite(y[k]);
        if (r < rows && !bad) continue;
        if (r < rows) {
#pragma nounroll
            for (int k = 0; k < E; ++k) {
                const T one = v[x * E + k];
                if (!not_finite(one)) continue;
                const int d = (x % (kHd / E)) * E + k;
                // query row q: token min(q >> hg_shift, tokens_left - 1) of the tile, at first + that
#pragma nounroll
                for (int q = 0; q < kPagedTileRows; ++q)
                    if (r <= first + min(q >> hg_shift, tokens_left - 1)) atomicOr(&poison[q][d >> 5], 1u << (d & 31));
                v[x * E + k] = (T)0.0f;
            }
        } else {
#pragma unroll
            for (int k = 0; k < E; ++k) y[k] = (T)0.0f;
            *reinterpret_cast<vec*>(v + x * E) = y;
        }
    }
}

// Four waves, two workgroups a CU: one computes while the other's rows arrive or
// its exponentials run.  Wave (rg, half) has query rows 32 rg .. and half of the
// 256 dims: it forms the scores' sums over its dims, exchanges them with its
// partner through LDS, takes the exponentials of all 32 cache rows of a step
// (both partners the same ones) and adds to its dims of the output.  So a wave
// holds half of a row's q (64 registers) and half of its output (64), two waves
// fit a SIMD, and each K and V value is read from LDS by two waves.
// 32 x 32 x 16 instructions on fp16 with the fp32 operands q and P as two fp16
// values each: hi + lo, 22 bits, two products an operand pair.  K and V steps of
// 32 rows come to LDS by loads that bypass the registers, K once the step's
// scores are formed, V into a second buffer.  K's 16-byte chunks are permuted by
// row (chunk ^ row % 16) so that the 32 rows a read touches fall into different
// banks; V rows are read as they are and transposed in registers (8 rows x 4
// dims a lane).  q rows come, and output rows go, through LDS too, a row a wave
// at a time (32 rows an instruction took 10 us a tile).
constexpr int kStep = 32;                 // cache rows of a step

__global__ __launch_bounds__(NT, 2) void paged_prefill_f16(PagedView pv, PagedBatch b, const float* __restrict__ q_gate,
                                                           const float* __restrict__ q_norm, float* __restrict__ out,
                                                           float* __restrict__ part_o, float* __restrict__ part_ml,
                                                           int hg_shift, int ng, float eps) {
    // One block of 64 KiB: K and V of the steps and the exchanged scores, or the
    // tile's 64 rows of q or of the output.
    struct Steps {
        _Float16 k[kStep][kHd], v[2][kStep][kHd];
        float4 x[4][4][kWave];
    };
    __shared__ __align__(16) char smem[sizeof(Steps)];
    static_assert(sizeof(Steps) == kPagedTileRows * kHd * sizeof(float), "the rows take the block's place");
    __shared__ uint32_t poison[kPagedTileRows][kHd / 32];
    Steps& st = *reinterpret_cast<Steps*>(smem);
    float4* const tile = reinterpret_cast<float4*>(smem);         // [64][64] 16-byte chunks, chunk ^ row % 32
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rg = wave & 1, half = wave >> 1;
    const int nn = lane & 31, h = lane >> 5;
    const int hg = 1 << hg_shift, tm = kPagedTileRows >> hg_shift;
    const int groups = pv.nkv * ng, nh = groups << hg_shift;
    const int wg = xcd_remap(blockIdx.x, gridDim.x);      // neighbours, which share K and V, on one XCD's L2
    const uint32_t kaddr = lds_address(&st.k[8 * wave][0]), vaddr = lds_address(&st.v[0][8 * wave][0]);

    const int qe = q_exponent(q_norm, lane);
    const float up = ldexpf(1.0f, qe), down = ldexpf(1.0f, -qe);
    const Units un = units_of(pv, b, groups, hg_shift, lane);
    Walk wk;
    wk.begin(un, wg, gridDim.x);
    while (wk.next(b, un, groups, hg_shift)) {
        const int seq = b.seq[wk.i], kvh = wk.y / ng;
        const int* table = pv.table + (size_t)seq * pv.max_pages;
        // Rows the tile's tokens see: [0, rows); the lane's query row sees [0, mine].
        const int rows = min(wk.start + min((wk.j + 1) * tm, wk.tokens), pv.max_rows);
        const int stop = min(rows, wk.t1 * kUnit), last16 = (rows - 1) & ~15;
        const int first = wk.start + wk.j * tm;            // position of the tile's first token
        // Query row r of the tile: token, and the row of q and out.
        auto token = [&](int r) { return wk.j * tm + (r >> hg_shift); };
        auto row_at = [&](int r) {
            return (size_t)(b.off[wk.i] + min(token(r), wk.tokens - 1)) * nh + (wk.y << hg_shift) + (r & (hg - 1));
        };
        const int mine = min(wk.start + min(token(32 * rg + nn), wk.tokens - 1), pv.max_rows - 1);

        // q rows to LDS.
#pragma unroll 4
        for (int r = 16 * wave; r < 16 * wave + 16; ++r)
            dma16(q_gate + row_at(r) * 2 * kHd + 4 * (lane ^ (r & 31)), lds_address(tile + r * (kHd / 4)));
        for (int x = tid; x < kPagedTileRows * (kHd / 32); x += NT) (&poison[0][0])[x] = 0;

        // A wave brings 8 rows of a step's K and V.  It holds 64 entries of the page
        // table, one a lane, from entry `held` on.
        int held = 0, ids = 0;
        auto hold = [&](int entry) {
            held = entry;
            ids = page_of(table, entry + lane, pv.max_pages, pv.n_pages);
        };
        auto row8 = [&](int base) { return min(base + 8 * wave, last16 + (8 * wave & 8)); };
        hold(row8(wk.t0 * kUnit) >> pv.page_shift);
        auto issue = [&](int base, int par) {
            const int r = row8(base), entry = r >> pv.page_shift;
            if (__builtin_expect(entry - held >= kWave, 0)) hold(entry);
            const size_t at = row_offset<_Float16>(pv, __builtin_amdgcn_readlane(ids, entry - held), kvh, r);
            const _Float16* kp = (const _Float16*)pv.k + at + h * kHd;
            const _Float16* vp = (const _Float16*)pv.v + at + 8 * lane;
            const int c0 = (lane & 31) ^ h ^ (8 * (wave & 1));
#pragma unroll
            for (int k = 0; k < 8; k += 2) dma16(kp + k * kHd + 8 * (c0 ^ k), kaddr + (uint32_t)(k * kHd * 2));
#pragma unroll
            for (int k = 0; k < 8; k += 2) dma16(vp + k * kHd, vaddr + (uint32_t)((par * kStep + k) * kHd * 2));
        };

        // q: lane (row nn, h) holds dims 128 half + 16 s + 8 h + j of its row: norm
        // (which the rotation leaves), then rotation, scale and the two halves.
        f16x8 qh[8], ql[8];
        {
            auto dims8 = [&](int c, float (&x)[8]) {       // chunks c, c + 1 of the lane's row
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float4 a = tile[(32 * rg + nn) * (kHd / 4) + ((c + k) ^ nn)];
                    x[4 * k] = a.x; x[4 * k + 1] = a.y; x[4 * k + 2] = a.z; x[4 * k + 3] = a.w;
                }
            };
            dma_wait();
            __syncthreads();
            float ss = 0.0f;
#pragma unroll 4
            for (int s = 0; s < 16; ++s) {
                float x[8];
                dims8(4 * s + 2 * h, x);
#pragma unroll
                for (int c = 0; c < 8; ++c) ss += x[c] * x[c];
            }
            const float scale = up * (kLog2e / 16.0f) / sqrtf(xor32_sum(ss) / (float)kHd + eps);
            const double* rope = pv.rope + (size_t)mine * kRopeDim + 8 * h;
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                float x[8], y[8];
                dims8(32 * half + 4 * s + 2 * h, x);
                if (half == 0 && s < 4) {                  // dims 16 (s % 2) + 8 h .. and 32 further
                    dims8(4 * (s ^ 2) + 2 * h, y);
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const float cs = (float)rope[16 * (s & 1) + c], sn = (float)rope[kRopeHalf + 16 * (s & 1) + c];
                        x[c] = s < 2 ? x[c] * cs - y[c] * sn : y[c] * sn + x[c] * cs;
                    }
                }
#pragma unroll
                for (int c = 0; c < 8; ++c) y[c] = x[c] * (scale * (1.0f + q_norm[128 * half + 16 * s + 8 * h + c]));
                split16(y, qh[s], ql[s]);
            }
        }

        f32x16 o[4];                                       // dims 128 half + 4 row + d at [d]
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int k = 0; k < 16; ++k) o[d][k] = 0.0f;
        float m_run = -INFINITY, l_run = 0.0f;

        __syncthreads();                                   // q is read
        int par = 0;
        if (wk.t0 * kUnit < stop) issue(wk.t0 * kUnit, 0);
        for (int base = wk.t0 * kUnit; base < stop; base += kStep) {
            dma_wait();
            __syncthreads();                               // the step's rows are there, the last one's V and scores read
            // Some row of the tile does not see some row of the step.
            const bool masked = base + kStep - 1 > first;
            if (masked)
                guard_rows(&st.v[par][8 * wave][0], 8, base + 8 * wave, rows, poison, first, wk.tokens - wk.j * tm,
                           hg_shift, lane);
            f32x16 sc;
#pragma unroll
            for (int k = 0; k < 16; ++k) sc[k] = 0.0f;
#pragma unroll
            for (int s = 0; s < 8; ++s) {                  // K operand: lane (row nn, h), dims 128 half + 16 s + 8 h ..
                const f16x8 a = *reinterpret_cast<const f16x8*>(&st.k[nn][8 * ((16 * half + 2 * s + h) ^ (nn & 15))]);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ql[s], sc, 0, 0, 0);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[s], sc, 0, 0, 0);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) st.x[wave][k][lane] = make_float4(sc[4 * k], sc[4 * k + 1], sc[4 * k + 2], sc[4 * k + 3]);
            lds_barrier();                                 // the scores are there, K is read
            if (base + kStep < stop) issue(base + kStep, par ^ 1);
            float mx = -INFINITY;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float4 y = st.x[wave ^ 2][k][lane];
                sc[4 * k] += y.x; sc[4 * k + 1] += y.y; sc[4 * k + 2] += y.z; sc[4 * k + 3] += y.w;
            }
            if (masked) {
                asm volatile("");                          // a branch: selects on every step cost more
                const int lim = mine - base - 4 * h;
#pragma unroll
                for (int k = 0; k < 16; ++k) sc[k] = 8 * (k >> 2) + (k & 3) <= lim ? sc[k] : -INFINITY;
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) mx = fmaxf(mx, sc[k]);
            mx = xor32_max(mx * down);
            if (__any(mx > m_run + kLazy)) {               // (m_run is -inf at first)
                const float m_new = fmaxf(m_run, mx);
                const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.0f : m_new));
                m_run = m_new;
                l_run *= alpha;
#pragma unroll
                for (int d = 0; d < 4; ++d) o[d] *= alpha;
            }
            const float sub = kPShift - (m_run == -INFINITY ? 0.0f : m_run);
            f16x8 ph[2], pl[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float p[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    p[k] = __builtin_amdgcn_exp2f(fmaf(sc[8 * c + k], down, sub));
                    l_run += p[k];
                }
                split16(p, ph[c], pl[c]);
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                // V rows 16 c + 4 h + {0..3, 8..11}: the weights' rows of the lane's half.
                const _Float16* vt = &st.v[par][16 * c + 4 * h][128 * half + 4 * nn];
                uint2 v8[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) v8[r] = *reinterpret_cast<const uint2*>(vt + ((r & 3) + 8 * (r >> 2)) * kHd);
#pragma unroll
                for (int d = 0; d < 4; ++d) {              // dims 4 m + d of the lane's 8 rows
                    const uint32_t sel = (d & 1) ? 0x07060302u : 0x05040100u;
                    u32x4 a;
#pragma unroll
                    for (int w = 0; w < 4; ++w)
                        a[w] = d < 2 ? __builtin_amdgcn_perm(v8[2 * w + 1].x, v8[2 * w].x, sel)
                                     : __builtin_amdgcn_perm(v8[2 * w + 1].y, v8[2 * w].y, sel);
                    const f16x8 av = __builtin_bit_cast(f16x8, a);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av, pl[c], o[d], 0, 0, 0);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av, ph[c], o[d], 0, 0, 0);
                }
            }
            par ^= 1;
        }

        // The tile's rows to LDS, then a row a wave at a time: finished, or as a part
        // to the workspace.  Both partners have the rows' sums.
        const bool whole = wk.t0 == 0 && wk.t1 == wk.tiles;
        const int slot = 2 * wg + (wk.t0 == 0);
        l_run = xor32_sum(l_run);
        const float inv = whole ? 1.0f / l_run : 1.0f;
        __syncthreads();                                   // V and the scores are read
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int chunk = 32 * half + 8 * (k >> 2) + 4 * h + (k & 3);
            tile[(32 * rg + nn) * (kHd / 4) + (chunk ^ nn)] =
                make_float4(o[0][k] * inv, o[1][k] * inv, o[2][k] * inv, o[3][k] * inv);
        }
        if (!whole && half == 0 && h == 0) {
            const size_t r = (size_t)slot * kPagedTileRows + 32 * rg + nn;
            part_ml[2 * r] = m_run;
            part_ml[2 * r + 1] = l_run;
        }
        __syncthreads();
#pragma unroll
        for (int k0 = 0; k0 < 16; k0 += 8) {
            float4 gate[8];
            if (whole) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    gate[k] = *reinterpret_cast<const float4*>(q_gate + row_at(16 * wave + k0 + k) * 2 * kHd + kHd + 4 * lane);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int r = 16 * wave + k0 + k;
                float4 x = tile[r * (kHd / 4) + (lane ^ (r & 31))];
                const uint32_t nan = poison[r][lane >> 3] >> (4 * (lane & 7));
                x.x = nan & 1 ? NAN : x.x;
                x.y = nan & 2 ? NAN : x.y;
                x.z = nan & 4 ? NAN : x.z;
                x.w = nan & 8 ? NAN : x.w;
                if (!whole)
                    *reinterpret_cast<float4*>(part_o + ((size_t)slot * kPagedTileRows + r) * kHd + 4 * lane) = x;
                else if (token(r) < wk.tokens)
                    *reinterpret_cast<float4*>(out + row_at(r) * kHd + 4 * lane) = gated(x, gate[k]);
            }
        }
        __syncthreads();
    }
}

// ---- fp32 cache -----------------------------------------------------------

constexpr int kF32Rows = 32;            // cache rows of an LDS tile (two tiles a unit)

// Four waves of 16 query rows each; fp32 instructions (16 x 16 x 4).  One LDS
// tile of K and V at a time, two workgroups a CU: one computes while the
// other's rows arrive.
__global__ __launch_bounds__(NT, 2) void paged_prefill_f32(PagedView pv, PagedBatch b, const float* __restrict__ q_gate,
                                                           const float* __restrict__ q_norm, float* __restrict__ out,
                                                           float* __restrict__ part_o, float* __restrict__ part_ml,
                                                           int hg_shift, int ng, float eps) {
    __shared__ __align__(16) float ks[kF32Rows][kHd], vs[kF32Rows][kHd];
    __shared__ uint32_t poison[kPagedTileRows][kHd / 32];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int hg = 1 << hg_shift, tm = kPagedTileRows >> hg_shift;
    const int groups = pv.nkv * ng, nh = groups << hg_shift;
    const int wg = xcd_remap(blockIdx.x, gridDim.x);

    const uint32_t kaddr = lds_address(&ks[8 * wave][0]), vaddr = lds_address(&vs[8 * wave][0]);

    const Units un = units_of(pv, b, groups, hg_shift, lane);
    Walk wk;
    wk.begin(un, wg, gridDim.x);
    while (wk.next(b, un, groups, hg_shift)) {
        const int seq = b.seq[wk.i], kvh = wk.y / ng;
        const int* table = pv.table + (size_t)seq * pv.max_pages;
        const int rows = min(wk.start + min((wk.j + 1) * tm, wk.tokens), pv.max_rows);
        const int at_tok = wk.j * tm + ((wave * 16 + n) >> hg_shift);
        const int tok = min(at_tok, wk.tokens - 1);
        const int mine = min(wk.start + tok, pv.max_rows - 1);
        const int head = (wk.y << hg_shift) + ((wave * 16 + n) & (hg - 1));
        const bool real = at_tok < wk.tokens;
        const size_t qrow = (size_t)(b.off[wk.i] + tok) * nh + head;
        const int last16 = (rows - 1) & ~15;

        __syncthreads();                           // the segment before has read its marks
        for (int x = tid; x < kPagedTileRows * (kHd / 32); x += NT) (&poison[0][0])[x] = 0;

        // q: lane (row n, g) holds dims 16 t + 4 g + c of its row.
        float q[64];
        {
            const float* qp = q_gate + qrow * 2 * kHd + 4 * g;
            const double* rope = pv.rope + (size_t)mine * kRopeDim + 4 * g;
            float ss = 0.0f;
#pragma unroll
            for (int t = 0; t < 16; ++t) {
                const float4 a = *reinterpret_cast<const float4*>(qp + 16 * t);
                q[4 * t] = a.x; q[4 * t + 1] = a.y; q[4 * t + 2] = a.z; q[4 * t + 3] = a.w;
            }
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float cs = (float)rope[16 * t + c], sn = (float)rope[kRopeHalf + 16 * t + c];
                    const float lo = q[4 * t + c], hi = q[4 * t + 8 + c];
                    q[4 * t + c] = lo * cs - hi * sn;
                    q[4 * t + 8 + c] = lo * sn + hi * cs;
                }
#pragma unroll
            for (int k = 0; k < 64; ++k) ss += q[k] * q[k];
            const float scale = kLog2e / 16.0f / sqrtf(xor16_sum(xor32_sum(ss)) / (float)kHd + eps);
#pragma unroll
            for (int t = 0; t < 16; ++t) {
                const float4 w = *reinterpret_cast<const float4*>(q_norm + 16 * t + 4 * g);
                q[4 * t] *= scale * (1.0f + w.x);
                q[4 * t + 1] *= scale * (1.0f + w.y);
                q[4 * t + 2] *= scale * (1.0f + w.z);
                q[4 * t + 3] *= scale * (1.0f + w.w);
            }
        }

        f32x4 o[16];            // dims 64 t + 4 (4 g + i) + c at [4 t + c][i]
#pragma unroll
        for (int x = 0; x < 16; ++x) o[x] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m_run = -INFINITY, l_run = 0.0f;

        const int stop = min(rows, wk.t1 * kUnit);
        for (int base = wk.t0 * kUnit; base < stop; base += kF32Rows) {
            __syncthreads();                       // the tile before is read
            {
                const int r = min(base + 8 * wave, last16 + (8 * wave & 8));   // 8 rows a wave, in one 16-row group
                const int page = page_of(table, r >> pv.page_shift, pv.max_pages, pv.n_pages);
                const size_t at = row_offset<float>(pv, page, kvh, r);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    dma16((const float*)pv.k + at + k * kHd + 4 * (lane ^ ((8 * wave + k) & 15)), kaddr + k * kHd * 4);
#pragma unroll
                for (int k = 0; k < 8; ++k) dma16((const float*)pv.v + at + k * kHd + 4 * lane, vaddr + k * kHd * 4);
            }
            dma_wait();
            __syncthreads();
            const bool masked = base + kF32Rows - 1 > wk.start + wk.j * tm;
            if (masked) {
                guard_rows(&vs[8 * wave][0], 8, base + 8 * wave, rows, poison, wk.start + wk.j * tm,
                           wk.tokens - wk.j * tm, hg_shift, lane);
                lds_barrier();
            }
            f32x4 sa[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int t = 0; t < 16; ++t) {
                f32x4 kf[2];
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
                    kf[kb] = *reinterpret_cast<const f32x4*>(&ks[16 * kb + n][4 * ((4 * t + g) ^ n)]);
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
                        sa[kb] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[kb][c], q[4 * t + c], sa[kb], 0, 0, 0);
            }
            float s[8], mx = -INFINITY;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                s[k] = sa[k >> 2][k & 3];
                if (masked) s[k] = base + 16 * (k >> 2) + 4 * g + (k & 3) <= mine ? s[k] : -INFINITY;
                mx = fmaxf(mx, s[k]);
            }
            mx = xor16_max(xor32_max(mx));
            if (__any(mx > m_run + kLazy)) {
                const float m_new = fmaxf(m_run, mx);
                const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.0f : m_new));
                m_run = m_new;
                l_run *= alpha;
#pragma unroll
                for (int x = 0; x < 16; ++x) o[x] *= alpha;
            }
            const float sub = m_run == -INFINITY ? 0.0f : m_run;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                s[k] = __builtin_amdgcn_exp2f(s[k] - sub);
                l_run += s[k];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const f32x4 x = *reinterpret_cast<const f32x4*>(&vs[16 * (k >> 2) + 4 * g + (k & 3)][64 * t + 4 * n]);
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        o[4 * t + c] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[c], s[k], o[4 * t + c], 0, 0, 0);
                }
        }
        __syncthreads();

        l_run = xor16_sum(xor32_sum(l_run));
        const bool whole = wk.t0 == 0 && wk.t1 == wk.tiles;
        const int slot = 2 * wg + (wk.t0 == 0);
        const size_t prow = (size_t)slot * kPagedTileRows + 16 * wave + n;
        const float inv = 1.0f / l_run;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = 64 * t + 4 * (4 * g + i);
                float4 x = make_float4(o[4 * t][i], o[4 * t + 1][i], o[4 * t + 2][i], o[4 * t + 3][i]);
                const uint32_t nan = poison[16 * wave + n][at >> 5] >> (at & 31);
                if (nan & 1) x.x = NAN;
                if (nan & 2) x.y = NAN;
                if (nan & 4) x.z = NAN;
                if (nan & 8) x.w = NAN;
                if (!whole) {
                    *reinterpret_cast<float4*>(part_o + prow * kHd + at) = x;
                } else if (real) {
                    const float4 gt = *reinterpret_cast<const float4*>(q_gate + qrow * 2 * kHd + kHd + at);
                    *reinterpret_cast<float4*>(out + qrow * kHd + at) =
                        gated(make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv), gt);
                }
            }
        if (!whole && g == 0) {
            part_ml[2 * prow] = m_run;
            part_ml[2 * prow + 1] = l_run;
        }
    }
}

// ---- joining cut tiles ------------------------------------------------------

// 16 query rows of one tile a workgroup, where the tile's units went to several
// workgroups: a wave four rows, a lane four dims.
__global__ __launch_bounds__(NT) void paged_prefill_merge(PagedView pv, PagedBatch b, const float* __restrict__ part_o,
                                                          const float* __restrict__ part_ml,
                                                          const float* __restrict__ q_gate, float* __restrict__ out,
                                                          int hg_shift, int ng, int nwg) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int groups = pv.nkv * ng, nh = groups << hg_shift, tm = kPagedTileRows >> hg_shift;
    const Units un = units_of(pv, b, groups, hg_shift, lane);
    const long per = (un.total + nwg - 1) / nwg;
    // The workgroup's tile: the sequences' tiles in order.
    int tile_end = lane < b.n ? ((b.off[lane + 1] - b.off[lane] + tm - 1) / tm) * groups : 0;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int x = __shfl_up(tile_end, o, kWave);
        if (lane >= o) tile_end += x;
    }
    const int q = blockIdx.x >> 2;
    const int i = __popcll(__ballot(tile_end <= q));
    const int tokens = b.off[i + 1] - b.off[i];
    const Tiles ts(__builtin_amdgcn_readlane(un.start, i), tokens, hg_shift);
    const int local = q - (__builtin_amdgcn_readlane(tile_end, i) - ts.n * groups);
    const int y = local / ts.n, o = local - y * ts.n, j = ts.tile(o);
    const long each = ts.before(ts.n);
    const long s = readlane_long(un.end, i) - each * groups + y * each + ts.ordered(o);
    const int w0 = (int)(s / per), w1 = (int)((s + ts.cnt(j) - 1) / per);
    if (w0 == w1) return;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int row = (blockIdx.x & 3) * 16 + wave * 4 + r;
        const int tok = j * tm + (row >> hg_shift);
        if (tok >= tokens) continue;
        const size_t qrow = (size_t)(b.off[i] + tok) * nh + (y << hg_shift) + (row & ((1 << hg_shift) - 1));
        const float4 gt = *reinterpret_cast<const float4*>(q_gate + qrow * 2 * kHd + kHd + 4 * lane);
        auto part = [&](int w) { return (size_t)(2 * w + (w == w0)) * kPagedTileRows + row; };
        float M = -INFINITY;
        for (int w = w0 + lane; w <= w1; w += kWave) M = fmaxf(M, part_ml[2 * part(w)]);
        M = wave_max(M);
        const float mu = M == -INFINITY ? 0.0f : M;
        float l = 0.0f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        constexpr int U = 4;
        for (int w = w0; w <= w1; w += U) {
            float4 p[U];
            float e[U], ls[U];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const size_t at = part(min(w + k, w1));
                p[k] = reinterpret_cast<const float4*>(part_o + at * kHd)[lane];
                e[k] = part_ml[2 * at];
                ls[k] = part_ml[2 * at + 1];
            }
#pragma unroll
            for (int k = 0; k < U; ++k) {
                if (w + k > w1) break;
                // a part none of whose rows this row sees has maximum -inf
                const float f = __builtin_amdgcn_exp2f(e[k] - mu);
                l += f * ls[k];
                x.x += f * p[k].x; x.y += f * p[k].y; x.z += f * p[k].z; x.w += f * p[k].w;
            }
        }
        const float inv = 1.0f / l;
        *reinterpret_cast<float4*>(out + qrow * kHd + 4 * lane) =
            gated(make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv), gt);
    }
}

// Two workgroups a CU.
int prefill_workgroups(const q35m_ctx* c) { return 2 * c->n_cu; }

}  // namespace

size_t paged_prefill_work_bytes(const q35m_ctx* c) {
    return (size_t)2 * prefill_workgroups(c) * kPagedTileRows * (kHd + 2) * sizeof(float);
}

hipError_t launch_paged_prefill(q35m_paged* p, int layer, const PagedBatch& b, const float* q_gate, float* out) {
    q35m_ctx* c = p->ctx;
    const int per_kv = c->d.nh / c->d.nkv;
    const int hg = per_kv <= 16 ? per_kv : per_kv % 16 == 0 ? 16 : 8;
    const int ng = per_kv / hg, nwg = prefill_workgroups(c), tm = kPagedTileRows / hg;
    int hg_shift = 0;
    while ((1 << hg_shift) < hg) ++hg_shift;
    float* part_o = p->work;
    float* part_ml = part_o + (size_t)2 * nwg * kPagedTileRows * kHd;
    const PagedView pv = p->view(layer);
    const AttnLayer& L = c->full[layer];
    long tiles = 0;
    for (int i = 0; i < b.n; ++i) tiles += (long)(b.off[i + 1] - b.off[i] + tm - 1) / tm * c->d.nkv * ng;
    {
        ProfScope ps(c, K_PAGED_PREFILL);
        auto go = [&](auto kern) {
            hipExtLaunchKernelGGL(kern, dim3(nwg), dim3(NT), 0, c->stream, ps.a, ps.b, 0, pv, b, q_gate, L.q_norm, out,
                                  part_o, part_ml, hg_shift, ng, c->d.eps);
        };
        if (p->type == Q35M_KV_F16) go(paged_prefill_f16);
        else go(paged_prefill_f32);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    ProfScope ps(c, K_PAGED_PREFILL_MERGE);
    hipExtLaunchKernelGGL(paged_prefill_merge, dim3((unsigned)(4 * tiles)), dim3(NT), 0, c->stream, ps.a, ps.b, 0, pv, b,
                          part_o, part_ml, q_gate, out, hg_shift, ng, nwg);
    return hipGetLastError();
}

}  // namespace q35
