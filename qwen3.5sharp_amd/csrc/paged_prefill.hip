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
// is S^T's own register layout, so weights cross no lanes (the two waves that share
// query rows pass them on, or the halves of the scores, in that layout), and the
// softmax's statistics of a query row are registers of its lanes.
#include <algorithm>

#include "paged_device.h"

namespace q35 {
namespace {

constexpr int NT = 256;
constexpr int kUnit = 64;               // cache rows of a unit
constexpr float kLog2e = 1.4426950408889634f;

// ---- the units of a call ------------------------------------------------

// Query tiles of one (sequence, head group) and their units.  Tile j (TM = 64 /
// hg tokens) has cnt(j) = ceil((start + (j + 1) TM) / 64) units (the last tile,
// if short, may count one more than it has rows for), which is
// floor((q0 + j) / hg); sums of such floors are closed forms.
struct Tiles {
    int shift;             // log2 of tiles a unit
    int n;                 // tiles
    long q0;
    // more: log2 of what a unit is over 64 rows.
    __device__ __forceinline__ Tiles(int start, int tokens, int hg_shift, int more) : shift(hg_shift + more) {
        const int tm_shift = 6 - hg_shift, tm = 1 << tm_shift;
        n = (tokens + tm - 1) >> tm_shift;
        q0 = ((long)start + tm + (kUnit << more) - 1) >> tm_shift;
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
    int start, more;
    long end, total;
};
__device__ __forceinline__ Units units_of(const PagedView& pv, const PagedBatch& b, int groups, int hg_shift, int more,
                                          int lane) {
    Units u;
    u.start = 0;
    u.end = 0;
    const int tokens = lane < b.n ? b.off[lane + 1] - b.off[lane] : 0;
    u.more = more;
    if (lane < b.n) {
        u.start = pv.lens[b.seq[lane]];
        const Tiles t(u.start, tokens, hg_shift, u.more);
        u.end = t.before(t.n) * groups;
    }
    for (int o = 1; o < b.n; o <<= 1) {
        const long x = shfl_up_long(u.end, o);
        if (lane >= o) u.end += x;
    }
    u.end = lane < b.n ? u.end : readlane_long(u.end, b.n - 1);
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
            const Tiles ts(start, tokens, hg_shift, un.more);
            n = ts.n;
            const long each = ts.before(n);
            long rest = u - (readlane_long(un.end, i) - each * groups);
            y = (int)(rest / each);
            rest -= (long)y * each;
            // The last place whose units begin at or before rest: 64 places a step.
            const int lane = threadIdx.x & (kWave - 1);
            o = 0;
            for (int left = n; left > 1;) {              // among places [o, o + left)
                const int step = (left + kWave - 1) / kWave, c = lane * step;
                const int hits = __popcll(__ballot(c < left && ts.ordered(o + c) <= rest));
                o = uniform(o + (hits - 1) * step);
                left = uniform(min(step, left - (hits - 1) * step));
            }
            within = rest - ts.ordered(o);
        }
        const Tiles ts(start, tokens, hg_shift, un.more);
        y = uniform(y);
        o = uniform(o);
        n = uniform(n);
        j = ts.tile(o);
        tiles = uniform((int)ts.cnt(j));
        t0 = uniform((int)within);
        t1 = uniform((int)min((long)tiles, within + (u_end - u)));
        u = uniform(u + t1 - t0);
        if (un.more) t1 = tiles = uniform((int)Tiles(start, tokens, hg_shift, 0).cnt(j));      // a whole tile, in 64s
        return true;
    }
};

// ---- loads, and rows that not every query sees ----------------------------

// Loads straight to LDS (dma_nth below): 16 bytes a lane, to address at + 16 lane.
// Complete once vmcnt says so: dma_wait() before the barrier that publishes the
// rows.  The instruction is written out because the compiler, told of it, waits for
// all such loads before the next LDS read, also one of the other buffer.
__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(const lds_void*)p; }
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// V rows of a unit that not every query row of the tile sees.  Rows past the
// tile's last row hold anything and become zeros; a value that is not finite
// becomes zero too (0 x inf is NaN in the products of the query rows that do not
// see it), and `found` is set, upon which the outputs of the query rows that do are
// settled at the segment's end.  A wave takes COUNT rows of kHd values from v on;
// base: their first row's position.  (Rows up to `first` are seen by all of the tile.)
// The top bit of each value's place set where it is not finite: its exponent plus
// one, of 32 bits of values.
template <typename T>
__device__ __forceinline__ uint32_t full_exponents(uint32_t x) {
    return sizeof(T) == 2 ? (x & 0x7c007c00u) + 0x04000400u : (x & 0x7f800000u) + 0x00800000u;
}
template <int COUNT, typename T>
__device__ __forceinline__ void guard_rows(T* v, int base, int rows, int* found, int first, int lane) {
    constexpr int E = 16 / sizeof(T);          // values of 16 bytes
    typedef T vec __attribute__((ext_vector_type(E)));
    if (base >= rows) {
#pragma unroll
        for (int x = 0; x < COUNT * (kHd / E); x += kWave) *reinterpret_cast<vec*>(v + (x + lane) * E) = vec{};
        return;
    }
    constexpr int count = COUNT, U = 4;        // U chunks a lane looks at together
#pragma nounroll
    for (int x0 = max(0, first + 1 - base) * (kHd / E) + lane; x0 < count * (kHd / E); x0 += U * kWave) {
        u32x4 y[U];
#pragma unroll
        for (int u = 0; u < U; ++u) y[u] = *reinterpret_cast<u32x4*>(v + min(x0 + u * kWave, count * (kHd / E) - 1) * E);
        uint32_t full = 0;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k) full |= full_exponents<T>(y[u][k]);
        const int end = base + min(x0 + (U - 1) * kWave, count * (kHd / E) - 1) / (kHd / E);     // the last one's row
        if (end < rows && !(full & (sizeof(T) == 2 ? 0x80008000u : 0x80000000u))) continue;
#pragma nounroll
        for (int x = x0; x < min(x0 + U * kWave, count * (kHd / E)); x += kWave) {
            if (base + x / (kHd / E) >= rows) {
                *reinterpret_cast<vec*>(v + x * E) = vec{};
                continue;
            }
#pragma nounroll
            for (int k = 0; k < E; ++k)
                if (not_finite(v[x * E + k])) {
                    v[x * E + k] = (T)0.0f;
                    *found = 1;
                }
        }
    }
}

// ---- a segment's beginning and end, one row of four waves' tile a lane -------

// Half of a q row, of which LDS has the fp32 values at `at` (16-byte chunks ^ row %
// 32) once every wave's loads are there: x[s] is dims 128 half + 16 s + 8 h .. of
// row 32 rg + lane % 32, rotated; returned is what makes it the norm's row over 16
// in powers of two.  ss: room for four waves' sums.
__device__ __forceinline__ float q_row(float (&x)[8][8], const float4* at, const double* rope, float (*ss_of)[32], int rg,
                                       int half, int lane, float eps) {
    const int nn = lane & 31, h = lane >> 5;
    double cs[16], sn[16];
    if (half == 0) {
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            cs[k] = rope[8 * h + (k & 8) * 2 + (k & 7)];
            sn[k] = rope[kRopeHalf + 8 * h + (k & 8) * 2 + (k & 7)];
        }
    }
    dma_wait();
    __syncthreads();
    float ss = 0.0f;
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const float4 a = at[(32 * half + 4 * s + 2 * h + c) ^ nn];
            x[s][4 * c] = a.x; x[s][4 * c + 1] = a.y; x[s][4 * c + 2] = a.z; x[s][4 * c + 3] = a.w;
            ss += a.x * a.x; ss += a.y * a.y; ss += a.z * a.z; ss += a.w * a.w;
        }
    ss = xor32_sum(ss);
    if (h == 0) ss_of[2 * half + rg][nn] = ss;
    if (half == 0) {
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const float lo = x[k >> 3][k & 7], hi = x[2 + (k >> 3)][k & 7];
            x[k >> 3][k & 7] = lo * (float)cs[k] - hi * (float)sn[k];
            x[2 + (k >> 3)][k & 7] = lo * (float)sn[k] + hi * (float)cs[k];
        }
    }
    lds_barrier();                                         // (the raw values are read, too)
    return kLog2e / 16.0f / sqrtf((ss_of[rg][nn] + ss_of[rg + 2][nn]) / (float)kHd + eps);
}

// Wave (rg, half)'s output, dims 128 half + 32 d + (its register's row) of query row
// 32 rg + lane % 32 at [d], to LDS, 16-byte chunks ^ row % 32.
__device__ __forceinline__ void put_rows(float4* os, const f32x16 (&o)[4], int rg, int half, int lane) {
    const int nn = lane & 31, h = lane >> 5;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int k = 0; k < 16; k += 4)
            os[(32 * rg + nn) * (kHd / 4) + ((32 * half + 8 * d + 2 * (k >> 2) + h) ^ nn)] =
                make_float4(o[d][k], o[d][k + 1], o[d][k + 2], o[d][k + 3]);
}

// From there a wave's 16 rows leave, one at a time: finished to out_row(row), the
// lane's place (none if null), or as parts.  l, m: sum and maximum of row 16 wave + lane % 16.
// Whether a value of theirs is not finite.
template <typename F>
__device__ __forceinline__ bool leave_rows(const float4* os, float l, float m, bool whole, float4 (&gate)[16], float* part_o,
                                           float* part_ml, int wave, int lane, F out_row) {
    float nan[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    auto rows8 = [&](int k0, auto&& put) {
        float4 x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int r = 16 * wave + k0 + k;
            x[k] = os[r * (kHd / 4) + (lane ^ (r & 31))];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            nan[0] = fmaf(x[k].x, 0.0f, nan[0]); nan[1] = fmaf(x[k].y, 0.0f, nan[1]);
            nan[2] = fmaf(x[k].z, 0.0f, nan[2]); nan[3] = fmaf(x[k].w, 0.0f, nan[3]);
            put(k0 + k, x[k]);
        }
    };
    if (whole) {
        const float inv_l = 1.0f / l;
        // (all gates before the first store: a wait for a load waits for the stores before it)
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            gate[k] = gate_sigmoid(gate[k]);
            asm volatile("" : "+v"(gate[k].x), "+v"(gate[k].y), "+v"(gate[k].z), "+v"(gate[k].w));
        }
        auto put = [&](int k, float4 x) {
            const float inv = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, inv_l), k));
            const float4 g = gate[k];
            x = make_float4(x.x * inv * g.x, x.y * inv * g.y, x.z * inv * g.z, x.w * inv * g.w);
            if (char* to = out_row(16 * wave + k)) *reinterpret_cast<float4*>(to) = x;
        };
        rows8(0, put);
        rows8(8, put);
    } else {
        float4* const po = reinterpret_cast<float4*>(part_o + 16 * wave * kHd);
        auto put = [&](int k, float4 x) { po[k * (kHd / 4) + lane] = x; };
        rows8(0, put);
        rows8(8, put);
        if (lane < 16) reinterpret_cast<float2*>(part_ml)[16 * wave + lane] = make_float2(m, l);
    }
    return __any((nan[0] + nan[1]) + (nan[2] + nan[3]) != 0.0f);      // (0 x inf is NaN)
}

// The wave's rows once more, with the infinities that their tokens see among the
// segment's rows [from, to) (query row q: up to first + min(q >> hg_shift, left - 1)).
// gate_row(row): the lane's place of the gate.
template <typename T, typename G, typename F>
__device__ __forceinline__ void settle_rows(const float4* os, const PagedView& pv, const int* table, int kvh, int from,
                                            int to, int first, int left, int hg_shift, float l, bool whole, float* part_o,
                                            int wave, int lane, G gate_row, F out_row) {
    uint32_t found = 0;
#pragma nounroll
    for (int k = 0; k < 16; ++k) {
        const int q = 16 * wave + k, end = min(to, first + min(q >> hg_shift, left - 1) + 1);
        found |= infinite_rows<T>(pv, table, kvh, from, end, lane);
        from = max(from, end);
        float4 x = settled(os[q * (kHd / 4) + (lane ^ (q & 31))], found);
        if (whole) {
            const float inv = 1.0f / __shfl(l, k, kWave);
            x = gated(make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv), *reinterpret_cast<const float4*>(gate_row(q)));
            if (char* to_row = out_row(q)) *reinterpret_cast<float4*>(to_row) = x;
        } else {
            reinterpret_cast<float4*>(part_o + q * kHd)[lane] = x;
        }
    }
}

// ---- fp16 cache -----------------------------------------------------------

// Four waves, one a SIMD.  Wave (rg, half) has query rows 32 rg ..: it forms the
// scores and weights of the unit's cache rows 32 half .., hands its weights to
// its partner through LDS, and adds all 64 rows' values to output dims 128 half
// ..; so a row's q is in both waves' registers (128 of them) but its output in
// one's (64), and the two never have to be joined.
// 32 x 32 x 16 instructions on fp16 with the fp32 operands q and P as two fp16
// values each: hi + lo, to 2^-23 of the value, two products an operand pair (three parts
// would be half as many products again; one part is 2^-11 off).  K and V units
// are double-buffered in LDS by loads that bypass the registers, 16-byte chunks
// permuted by row so that the rows that one read touches fall into different
// banks (K: chunk ^ row % 16, V: chunk ^ 4 (row % 4)); V is transposed as it is
// read.  q rows come, and output rows go, through LDS too, a row a wave at a time
// (32 rows an instruction took 10 us a tile).
// The units are software-pipelined: a unit's exponentials run among the score
// products of the next one, whose K is there a unit ahead of its V, and its last
// eight products among the first K reads of the next.  Both partners keep one
// maximum a row that the weights refer to; the maxima of a unit's two halves meet
// with the weights of the unit before, and it moves only when a score passes it by
// kMove.
// What bounds it: issue.  The 64 matrix instructions of a unit and SIMD are 2048
// cycles, of the 3400 that it takes at 1.8 GHz: a single wave a SIMD issues everything
// in order, about four vector instructions in a matrix instruction's shadow (16.4 ns a
// product with up to 4, 22.9 with 6, 34 with 12), so what is the same every unit is a
// kept address, a scalar or an offset in the instruction, the loads of the next unit
// are spread over the score products (in one run of 16 they held the wave for 800
// cycles), and every LDS read is a step ahead.  (Closer feeding gains less than it
// counts: on random operands the pipe pulls the clock to 1.55 GHz, 20 ns a product or
// 1.3 us a unit, where zeros take 15.)  2048 rows over as many: 92 us; 512 over 16384:
// 265 to 268 us.  Two workgroups a CU with half the registers each, partners splitting
// the dims and exchanging scores (twice the exponentials): 133 and 318 us.
// A segment's beginning and end are 30000 cycles of it (40 % of a call of 2048 rows):
// partners form half of q each (9000 -> 5800 cycles), and the last rows' LDS reads and the gates come
// before the first store, whose end a later load's wait would wait for (16000 ->
// 7000).
struct F16Tile {
    _Float16 k[2][kUnit][kHd], v[2][kUnit][kHd];
    f16x8 p[4][4][kWave];                 // a wave's weights: operands (hi, lo) of its two 16-row steps
    float mx[2][4][32];                   // maxima of a unit's halves; at the end sums and maxima
    float w[kHd];                         // 1 + the norm's weights
    int found;                            // values that are not finite
};
typedef const __attribute__((address_space(3))) f16x8 lds_f16x8;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// The i-th of eight loads for 8 KiB: global memory from `from` on, LDS
// from `at` on, 1 KiB each; off: the lane's place in that KiB of global memory.
// (The offset in the instruction counts on both sides.)
template <int K>
__device__ __forceinline__ void dma_kib(const void* from, uint32_t off, uint32_t at) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3" ::"s"(at), "v"(off), "s"(from),
                 "n"(1024 * K)
                 : "memory");
}
__device__ __forceinline__ void dma_nth(int i, const void* from, uint32_t off, uint32_t at) {
    if (i & 4) at += 4096, from = (const char*)from + 4096;
    if ((i & 3) == 0) dma_kib<0>(from, off, at);
    if ((i & 3) == 1) dma_kib<1>(from, off, at);
    if ((i & 3) == 2) dma_kib<2>(from, off, at);
    if ((i & 3) == 3) dma_kib<3>(from, off, at);
}
// A pointer that all lanes have the same, as the compiler cannot see.
__device__ __forceinline__ const void* uniform(const void* p) {
    const uint64_t x = (uint64_t)p;
    return (const void*)((uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32 | (uint32_t)uniform((int)x));
}

__global__ __launch_bounds__(NT, 1) void paged_prefill_f16(PagedView pv, PagedBatch b, const float* __restrict__ q_gate,
                                                           const float* __restrict__ q_norm, float* __restrict__ out,
                                                           float* __restrict__ part_o, float* __restrict__ part_ml,
                                                           int hg_shift, int ng, int more, float eps) {
    // Weights are e^{s - m} 2^kShift, and m is behind the largest score by up to kMove
    // (in log2): below 2^15.9, in fp16's range, and in steps of 2^-24, 2^-30 of the largest
    // weight or finer.  Half a step, 2^-31, is less than what adding 16 rows to an fp32
    // sum rounds off a row (2^-25 / 16).  A smaller kMove scales the output more often:
    // 2048 rows 92.7 us at (7, 8), 90.4 here, 88.5 at (1, 14), whose steps lose rows 18
    // nats below the largest.
    constexpr float kShift = 6.0f, kMove = 9.9f;
    __shared__ __align__(16) F16Tile st;
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rg = wave & 1, half = wave >> 1;
    const int hg = 1 << hg_shift, tm = kPagedTileRows >> hg_shift;
    const int groups = pv.nkv * ng, nh = groups << hg_shift;
    const int wg = xcd_remap(blockIdx.x, gridDim.x);      // neighbours, which share K and V, on one XCD's L2
    constexpr int kBuf = kUnit * kHd * 2;                 // bytes of a buffer
    const uint32_t kaddr = lds_address(&st.k[0][16 * wave][0]), vaddr = lds_address(&st.v[0][16 * wave][0]);

    const float w = q_norm[tid];
    const int qe = q_exponent(q_norm, tid & 63);
    const float up = ldexpf(1.0f, qe), down = ldexpf(1.0f, -qe);
    const Units un = units_of(pv, b, groups, hg_shift, more, tid & 63);
    st.w[tid] = 1.0f + w;                                 // (read behind the first segment's first barrier)
    Walk wk;
    wk.begin(un, wg, gridDim.x);
    while (wk.next(b, un, groups, hg_shift)) {
        const int start = uniform(wk.start), tokens = uniform(wk.tokens);
        const int seq = b.seq[wk.i], kvh = wk.y / ng;
        const int* table = pv.table + (size_t)seq * pv.max_pages;
        // (the lane's own places as values of this segment: addresses made of them
        // would else be kept over all segments)
        int lane = tid & 63, nn = lane & 31;
        asm volatile("" : "+v"(lane), "+v"(nn));
        const int h = lane >> 5;
        // Rows the tile's tokens see: [0, rows); the lane's query row sees [0, mine].
        const int rows = uniform(min(start + min((wk.j + 1) * tm, tokens), pv.max_rows));
        const int last16 = (rows - 1) & ~15;
        const int first = uniform(start + wk.j * tm);          // position of the tile's first token
        const int mine = min(start + min(wk.j * tm + ((32 * rg + nn) >> hg_shift), tokens - 1), pv.max_rows - 1);
        // Query row r of the tile is row row0 + from_row0(r) of q and out (the last
        // token's for rows past the `left` tokens): a 64-bit base a tile and 32 bits from
        // there.
        const int left = uniform(tokens - wk.j * tm);
        const long row0 = uniform((long)(uniform(b.off[wk.i]) + wk.j * tm) * nh + (wk.y << hg_shift));
        const char* const q_tile = (const char*)uniform(q_gate + row0 * 2 * kHd);
        char* const out_tile = (char*)uniform(out + row0 * kHd);
        auto from_row0 = [&](int r) { return min(r >> hg_shift, left - 1) * nh + (r & (hg - 1)); };

        // A wave brings its 16 rows of a unit's K or V.  It holds 64 entries of the
        // page table, one a lane, from entry `held` on.
        int held = 0, ids = 0;
        auto hold = [&](int entry) {
            held = entry;
            ids = page_of(table, entry + lane, pv.max_pages, pv.n_pages);
        };
        hold(min(wk.t0 * kUnit + 16 * wave, last16) >> pv.page_shift);
        auto group_at = [&](int t) {
            const int r = uniform(min(t * kUnit + 16 * wave, last16)), entry = r >> pv.page_shift;
            if (__builtin_expect(uniform(entry - held) >= kWave, 0)) hold(entry);
            return row_offset<_Float16>(pv, __builtin_amdgcn_readlane(ids, uniform(entry - held)), kvh, r);
        };
        uint32_t ko[8], vo[2];
#pragma unroll
        for (int r = 0; r < 16; r += 2) ko[r / 2] = 512u * h + 16u * (nn ^ h ^ r);
#pragma unroll
        for (int r = 0; r < 4; r += 2) vo[r / 2] = 512u * h + 16u * (nn ^ (4 * (h + r)));
        auto issue_k = [&](int i, const void* from, int buf) { dma_nth(i, from, ko[i], kaddr + buf * kBuf); };
        auto issue_v = [&](int i, const void* from, int buf) { dma_nth(i, from, vo[i & 1], vaddr + buf * kBuf); };
        auto k_from = [&](size_t at) { return uniform((const _Float16*)pv.k + at); };
        auto v_from = [&](size_t at) { return uniform((const _Float16*)pv.v + at); };

        // q rows to where V will be, 16-byte chunks permuted by row (chunk ^ row % 32).
        const float4* const qs = reinterpret_cast<const float4*>(&st.v[0][0][0]);
#pragma unroll 4
        for (int r = 16 * wave; r < 16 * wave + 16; ++r)
            dma_nth(0, q_tile, from_row0(r) * (2 * kHd * 4) + 16 * (lane ^ (r & 31)),
                     lds_address(&st.v[0][0][0]) + r * kHd * 4);
        // Where the wave's rows of the next units lie: found a unit before they are asked for.
        const size_t at0 = group_at(wk.t0);
#pragma unroll
        for (int i = 0; i < 8; ++i) issue_k(i, k_from(at0), 0);
        size_t at1 = group_at(wk.t0 + 1), at2 = group_at(wk.t0 + 2);
        if (tid == 0) st.found = 0;

        // q: lane (row nn, h) forms dims 128 half + 16 s + 8 h + j of its row, s < 8:
        // norm (which the rotation leaves), rotation, scale and the two halves, which
        // take the raw values' place.
        {
            float4* const at = const_cast<float4*>(qs) + (32 * rg + nn) * (kHd / 4);
            float x[8][8];
            const float scale = up * q_row(x, at, pv.rope + (size_t)mine * kRopeDim, st.mx[0], rg, half, lane, eps);
            const float* const w = &st.w[128 * half + 8 * h];
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                float y[8];
#pragma unroll
                for (int c = 0; c < 8; c += 4) {
                    const float4 v = *reinterpret_cast<const float4*>(&w[16 * s + c]);
                    y[c] = x[s][c] * (scale * v.x);
                    y[c + 1] = x[s][c + 1] * (scale * v.y);
                    y[c + 2] = x[s][c + 2] * (scale * v.z);
                    y[c + 3] = x[s][c + 3] * (scale * v.w);
                }
                f16x8 hi, lo;
                split16(y, hi, lo);
                at[(32 * half + 4 * s + 2 * h) ^ nn] = __builtin_bit_cast(float4, hi);
                at[(32 * half + 4 * s + 2 * h + 1) ^ nn] = __builtin_bit_cast(float4, lo);
            }
            lds_barrier();
        }
        // Then lane (row nn, h) holds dims 16 s + 8 h + j, s < 16.
        f16x8 qh[16], ql[16];
#pragma unroll
        for (int s = 0; s < 16; ++s) {
            qh[s] = __builtin_bit_cast(f16x8, qs[(32 * rg + nn) * (kHd / 4) + ((4 * s + 2 * h) ^ nn)]);
            ql[s] = __builtin_bit_cast(f16x8, qs[(32 * rg + nn) * (kHd / 4) + ((4 * s + 2 * h + 1) ^ nn)]);
        }

        // The output stays in accumulation registers all along: pin() is a use there,
        // without which the compiler moves all of it to vector registers and back on
        // every unit, for the rare branch that scales it.
        f32x16 o[4];                                       // dims 128 half + 32 d + row at [d]
        auto pin = [&]() { asm volatile("" : "+a"(o[0]), "+a"(o[1]), "+a"(o[2]), "+a"(o[3])); };
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int k = 0; k < 16; ++k) o[d][k] = 0.0f;
        pin();
        float m_run = -INFINITY, l_run = 0.0f, mx = -INFINITY;
        float sc[16];                                      // the wave's scores of a unit, before `down`

        // K operands of the wave's 32 rows: lane (row nn, h), dims 16 s + 8 h ..; V
        // operands of 16 rows and 32 dims: lane (dim nn, h), rows 4 h + {0..3, 8..11},
        // which the transposing read gathers from lanes of 4 rows x 16 dims.
        uint32_t ka[8], va[2][4];
#pragma unroll
        for (int s = 0; s < 8; ++s) ka[s] = lds_address(&st.k[0][32 * half + nn][0]) + 16 * ((2 * s + h) ^ (nn & 15));
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            va[0][d] = lds_address(&st.v[0][32 * half + 4 * h + ((lane >> 2) & 3)][0]) + 32 * (8 * half + ((2 * d + ((lane >> 4) & 1)) ^ (2 * ((lane >> 2) & 3)))) +
                    8 * (lane & 3);
            va[1][d] = va[0][d] + (half ? -32 * 512 : 32 * 512);   // the partner's rows
        }
        auto k_at = [&](int s) { return *(lds_f16x8*)(uintptr_t)(ka[s & 7] + 256 * (s >> 3)); };
        // Score products, K read four steps ahead (the first four by begin()), with
        // beside(s) among the products of step s.
        f16x8 kk[4];
        f32x16 x;
        auto begin = [&]() {
#pragma unroll
            for (int s = 0; s < 4; ++s) kk[s] = k_at(s);
        };
        auto scores = [&](auto beside) {
#pragma unroll
            for (int k = 0; k < 16; ++k) x[k] = 0.0f;
#pragma unroll
            for (int s = 0; s < 16; ++s) {
                const f16x8 k = kk[s & 3];
                x = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[s], x, 0, 0, 0);
                beside(s);
                if (s + 4 < 16) kk[s & 3] = k_at(s + 4);
                x = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[s], x, 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto take = [&]() {
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                sc[k] = x[k];
                asm volatile("" : "+v"(sc[k]));            // moved once, to vector registers
            }
        };
        // Whether some row of the tile does not see some row of unit t.
        auto masked = [&](int t) { return t * kUnit + kUnit - 1 > first; };
        auto mask = [&](int t) {
            const int lim = mine - (t * kUnit + 32 * half) - 4 * h;
#pragma unroll
            for (int k = 0; k < 16; ++k) sc[k] = 8 * (k >> 2) + (k & 3) <= lim ? sc[k] : -INFINITY;
        };
        // Posts the maximum of the unit's scores.
        auto post = [&]() {
            mx = fmaxf(sc[0], sc[1]);
#pragma unroll
            for (int k = 2; k < 16; ++k) mx = fmaxf(mx, sc[k]);
            mx = xor32_max(mx * down);
            if (h == 0) st.mx[0][wave][nn] = mx;
        };
        // The row's maximum over both halves of the unit, which may move the one the
        // weights refer to (known a while before it is done).
        bool moves;
        float sub;                                         // what the weights' exponents have added
        auto meet = [&](float other) {
            mx = fmaxf(mx, other);
            moves = __any(mx > m_run + kMove);             // (m_run is -inf at first)
        };
        auto move = [&]() {
            if (__builtin_expect_with_probability(moves, 0, 0.99)) {
                const float m_new = fmaxf(m_run, mx);
                const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.0f : m_new));
                m_run = m_new;
                l_run *= alpha;
                pin();
#pragma unroll
                for (int d = 0; d < 4; ++d) o[d] *= alpha;
                pin();
            }
            sub = kShift - (m_run == -INFINITY ? 0.0f : m_run);
        };
        f16x8 ph[2], pl[2];
        float p_even = 0.0f, p_sum = 0.0f;                 // (of the unit: one small weight at a time would be lost
                                                           // beside a large sum)
        auto weight = [&](int k) {
            const float p = __builtin_amdgcn_exp2f(fmaf(sc[k], down, sub));
            p_sum = k ? p_sum + p : p;
            if (k == 15) l_run += p_sum;
            asm volatile("" : "+v"(p_sum));                 // here, among the products
            if (k & 1) {
                f16x2 hi, lo;
                split16(p_even, p, hi, lo);
                ph[k >> 3][(k & 7) - 1] = hi.x; ph[k >> 3][k & 7] = hi.y;
                pl[k >> 3][(k & 7) - 1] = lo.x; pl[k >> 3][k & 7] = lo.y;
            } else {
                p_even = p;
            }
        };
        auto hand_over = [&]() {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                st.p[wave][2 * c][lane] = ph[c];
                st.p[wave][2 * c + 1][lane] = pl[c];
            }
        };
        auto v_read = [&](int whose, int step, f16x8 (&v)[4]) {
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const uint32_t at = va[whose][d] + step * 16 * 512;
                const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)at);
                const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(at + 8 * 512));
                typedef short s16x8 __attribute__((ext_vector_type(8)));
                v[d] = __builtin_bit_cast(f16x8, s16x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]});
            }
        };
        auto add = [&](const f16x8 (&v)[4], f16x8 hi, f16x8 lo) {
#pragma unroll
            for (int d = 0; d < 4; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[d], lo, o[d], 0, 0, 0);
#pragma unroll
            for (int d = 0; d < 4; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[d], hi, o[d], 0, 0, 0);
        };

        lds_barrier();                                     // q is read
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            issue_v(i, v_from(at0), 0);
            issue_k(i, k_from(at1), 1);
        }
        begin();
        scores([](int) {});
        take();
        if (masked(wk.t0)) mask(wk.t0);
        post();
        int t = wk.t0, buf = 0;
        lds_barrier();
        meet(st.mx[0][wave ^ 2][nn]);
        // Output products of unit t: the wave's own 32 rows, whose first 16 rows of V
        // are read by now, then its partner's.  The last 16 rows' wait, read, for the
        // next unit's beginning.  behind() runs among the first products, ahead() with
        // the partner's maxima.
        f16x8 v0[4], v1[4], h1, l1;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            h1[k] = l1[k] = (_Float16)0.0f;
#pragma unroll
            for (int d = 0; d < 4; ++d) v1[d][k] = (_Float16)0.0f;
        }
        auto output = [&](auto behind, auto ahead) {
            hand_over();
            v_read(0, 1, v1);
            __builtin_amdgcn_sched_barrier(0);
            behind();
            __builtin_amdgcn_sched_barrier(0);
            lds_barrier();                                 // the partner's weights and maxima
            const float other = st.mx[0][wave ^ 2][nn];
            const f16x8 h0 = st.p[wave ^ 2][0][lane], l0 = st.p[wave ^ 2][1][lane];
            h1 = st.p[wave ^ 2][2][lane];
            l1 = st.p[wave ^ 2][3][lane];
            v_read(1, 0, v0);
            __builtin_amdgcn_sched_barrier(0);
            add(v1, ph[1], pl[1]);
            ahead(other);
            __builtin_amdgcn_sched_barrier(0);
            v_read(1, 1, v1);
            add(v0, h0, l0);
            __builtin_amdgcn_sched_barrier(0);
        };
        // What every unit begins with: its rows and maxima are there (and K of the next
        // unit), every wave is past the buffers that the next rows go to.
        auto guard = [&]() {
            if (masked(t)) {
                guard_rows<16>(&st.v[buf][16 * wave][0], t * kUnit + 16 * wave, rows, &st.found, first, lane);
                lds_barrier();
            }
        };
#pragma nounroll
        for (; t + 1 < wk.t1; ++t) {
            dma_wait();
            __syncthreads();
            const int flip = buf ? -kBuf : kBuf;
#pragma unroll
            for (int s = 0; s < 8; ++s) ka[s] += flip;
            begin();
            __builtin_amdgcn_sched_barrier(0);
            const void* const next_k = k_from(at2);
            const void* const next_v = v_from(at1);
            at1 = at2;
            at2 = group_at(t + 3);
            guard();
            add(v1, h1, l1);
            move();
            scores([&](int s) {
                weight(s);
                if (s < 8)
                    issue_k(s, next_k, buf);
                else
                    issue_v(s - 8, next_v, buf ^ 1);
                if (s == 12) v_read(0, 0, v0);
            });
            output(
                [&]() {
#pragma unroll
                    for (int d = 0; d < 4; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v0[d], pl[0], o[d], 0, 0, 0);
                    take();
                    if (masked(t + 1)) {
                        asm volatile("");                  // a branch, not selects
                        mask(t + 1);
                    }
#pragma unroll
                    for (int d = 0; d < 4; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v0[d], ph[0], o[d], 0, 0, 0);
                    post();
                },
                meet);
#pragma unroll
            for (int d = 0; d < 4; ++d) va[0][d] += flip, va[1][d] += flip;
            buf ^= 1;
        }
        dma_wait();
        __syncthreads();
        const bool whole = wk.t0 == 0 && wk.t1 == wk.tiles;
        float4 gate[16];                                   // of the wave's rows 16 wave ..
        if (whole) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
                gate[r] = *reinterpret_cast<const float4*>(
                    q_tile + (uint32_t)(from_row0(16 * wave + r) * (2 * kHd * 4) + 4 * kHd + 16 * lane));
        }
        guard();
        add(v1, h1, l1);
        move();
#pragma unroll
        for (int k = 0; k < 16; ++k) weight(k);
        v_read(0, 0, v0);
        output([&]() { add(v0, ph[0], pl[0]); }, [](float) {});
        add(v1, h1, l1);
        pin();

        // The tile's rows to LDS, then a row a wave at a time: finished, or as a part
        // to the workspace.  (Places again as values of this part: kept from the
        // segment's beginning they would be in registers all the while.)
        asm volatile("" : "+v"(lane), "+v"(nn));
        const int slot = 2 * wg + (wk.t0 == 0);
        l_run = xor32_sum(l_run);
        if (lane < 32) st.mx[1][wave][nn] = l_run;
        if (half == 0 && lane < 32) st.mx[0][rg][nn] = m_run;
        lds_barrier();                                     // K and V are read, the last maxima too
        float4* const os = reinterpret_cast<float4*>(&st.k[0][0][0]);
        put_rows(os, o, rg, half, lane);
        lds_barrier();
        const int row = 16 * wave + (lane & 15);           // a row's sum and maximum in lane row % 16
        const float l = st.mx[1][row >> 5][row & 31] + st.mx[1][2 + (row >> 5)][row & 31];
        float* const to_part = part_o + (size_t)slot * kPagedTileRows * kHd;
        auto gate_row = [&](int r) { return q_tile + (uint32_t)(from_row0(r) * (2 * kHd * 4) + 4 * kHd + 16 * lane); };
        auto out_row = [&](int r) { return r >> hg_shift < left ? out_tile + (uint32_t)(from_row0(r) * (kHd * 4) + 16 * lane) : nullptr; };
        const bool look = leave_rows(os, l, st.mx[0][row >> 5][row & 31], whole, gate, to_part,
                                     part_ml + (size_t)2 * slot * kPagedTileRows, wave, lane, out_row);
        if (__builtin_expect(look || uniform(st.found), 0))
            settle_rows<_Float16>(os, pv, table, kvh, wk.t0 * kUnit, min(rows, wk.t1 * kUnit), first, left, hg_shift, l, whole,
                            to_part, wave, lane, gate_row, out_row);
        lds_barrier();                                     // (the stores need no wait)
    }
}

// ---- fp32 cache -----------------------------------------------------------

// The shape of the fp16 kernel, on steps of 32 cache rows, with every fp32 operand
// as three bf16 values, 8 bits of its mantissa each (exact), and the six products
// of an operand pair that reach 2^-16 of it: 24 bits, with fp32's range, at six
// bf16 instructions, 192 cycles where the fp32 instruction takes 512 for the same
// 32 x 32 x 16.  Those instructions take what is below 2^-126 as 0, parts and
// products: weights being up to one, the largest at 2^-14 or more, an output is off by up
// to 2^-112 a row, so values below 2^-96 begin to lose bits.
// Wave (rg, half) has query rows 32 rg ..; partners split the dims: each forms the
// scores' products of dims 128 half .. and hands them to the other, both form the
// weights, and each adds the output dims 128 half ...
// K and V come as fp32, K with 16-byte chunks ^ row % 16 and V with chunk ^ 8
// (row / 4 % 2), and are cut up where they are read, 5.5 instructions a value, in
// each wave for its 32 query rows: 7.3 a product, in the shadow of which they are
// placed one stage a product (left to itself the compiler puts 40 in a row: 3050
// cycles for 48 products instead of 2390).  133 rows over 8000: 130 us, 1000 over
// as many: 72 us back to back; the kernel of fp32 instructions took 165 and 112.
constexpr int kStep = 32;
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef const __attribute__((address_space(3))) f32x4 lds_f32x4;
typedef const __attribute__((address_space(3))) float lds_float;
struct F32Tile {
    float k[2][kStep][kHd], v[2][kStep][kHd];
    float4 x[4][4][kWave];                // a wave's half of the scores
    float ss[4][32];                      // q's sums of squares; at the end sums and maxima
    float w[kHd];
    int found;
};

struct Cut3 {
    b16x8 hi, mid, lo;
};
__device__ __forceinline__ uint32_t bits(float x) { return __builtin_bit_cast(uint32_t, x); }
__device__ __forceinline__ uint32_t tops(float a, float b) {   // the upper halves of two
    return __builtin_amdgcn_perm(bits(b), bits(a), 0x07060302u);
}
// The three parts of eight values, in six stages of about as many instructions (the
// remainders by masks and subtractions: the dot product with (-1, 0) that would
// take half the instructions shares the matrix pipe, and doubles a product's time).
struct Cutter {
    float mid[2], lo[2];
    u32x4 p[3];
    __device__ __forceinline__ void value(const float (&y)[8], int j) {
        const float hi2 = __builtin_bit_cast(float, bits(y[j]) & 0xffffff00u);      // 16 bits of the mantissa
        lo[j & 1] = y[j] - hi2;
        mid[j & 1] = hi2 - __builtin_bit_cast(float, bits(y[j]) & 0xffff0000u);
    }
    __device__ __forceinline__ void pair(const float (&y)[8], int j) {
        p[0][j] = tops(y[2 * j], y[2 * j + 1]);
        p[1][j] = tops(mid[0], mid[1]);
        p[2][j] = tops(lo[0], lo[1]);
    }
    __device__ __forceinline__ void stage(const float (&y)[8], int i) {
        const int j = 4 * (i / 3);
        if (i % 3 == 0) value(y, j), value(y, j + 1);
        if (i % 3 == 1) pair(y, j / 2), value(y, j + 2);
        if (i % 3 == 2) value(y, j + 3), pair(y, j / 2 + 1);
    }
    __device__ __forceinline__ Cut3 done() const {
        return {__builtin_bit_cast(b16x8, p[0]), __builtin_bit_cast(b16x8, p[1]), __builtin_bit_cast(b16x8, p[2])};
    }
};
__device__ __forceinline__ Cut3 cut3(const float (&y)[8]) {
    Cutter c;
#pragma unroll
    for (int i = 0; i < 6; ++i) c.stage(y, i);
    return c.done();
}
// c += a b, the small products first, with beside(i) behind the i-th.
template <typename F>
__device__ __forceinline__ f32x16 mul6(const Cut3& a, const Cut3& b, f32x16 c, F beside) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.lo, b.hi, c, 0, 0, 0);
    beside(0);
    __builtin_amdgcn_sched_barrier(0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.hi, b.lo, c, 0, 0, 0);
    beside(1);
    __builtin_amdgcn_sched_barrier(0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.mid, b.mid, c, 0, 0, 0);
    beside(2);
    __builtin_amdgcn_sched_barrier(0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.mid, b.hi, c, 0, 0, 0);
    beside(3);
    __builtin_amdgcn_sched_barrier(0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.hi, b.mid, c, 0, 0, 0);
    beside(4);
    __builtin_amdgcn_sched_barrier(0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.hi, b.hi, c, 0, 0, 0);
    beside(5);
    __builtin_amdgcn_sched_barrier(0);
    return c;
}

__global__ __launch_bounds__(NT, 1) void paged_prefill_f32(PagedView pv, PagedBatch b, const float* __restrict__ q_gate,
                                                           const float* __restrict__ q_norm, float* __restrict__ out,
                                                           float* __restrict__ part_o, float* __restrict__ part_ml,
                                                           int hg_shift, int ng, int more, float eps) {
    // Weights are e^{s - m} with m up to kMove (in log2) above the largest score: at most
    // one, so that an output overflows only where the sum of |V| over the rows does.
    constexpr float kMove = 14.0f;
    __shared__ __align__(16) F32Tile st;
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rg = wave & 1, half = wave >> 1;
    const int hg = 1 << hg_shift, tm = kPagedTileRows >> hg_shift;
    const int groups = pv.nkv * ng, nh = groups << hg_shift;
    const int wg = xcd_remap(blockIdx.x, gridDim.x);
    constexpr int kBuf = kStep * kHd * 4;                 // bytes of a buffer
    const uint32_t kaddr = lds_address(&st.k[0][8 * wave][0]), vaddr = lds_address(&st.v[0][8 * wave][0]);

    st.w[tid] = 1.0f + q_norm[tid];                       // (read behind the first segment's first barrier)
    const Units un = units_of(pv, b, groups, hg_shift, more, tid & 63);
    Walk wk;
    wk.begin(un, wg, gridDim.x);
    while (wk.next(b, un, groups, hg_shift)) {
        const int start = uniform(wk.start), tokens = uniform(wk.tokens);
        const int seq = b.seq[wk.i], kvh = wk.y / ng;
        const int* table = pv.table + (size_t)seq * pv.max_pages;
        int lane = tid & 63, nn = lane & 31;
        asm volatile("" : "+v"(lane), "+v"(nn));
        const int h = lane >> 5;
        const int rows = uniform(min(start + min((wk.j + 1) * tm, tokens), pv.max_rows));
        const int last16 = (rows - 1) & ~15;
        const int first = uniform(start + wk.j * tm);     // position of the tile's first token
        const int mine = min(start + min(wk.j * tm + ((32 * rg + nn) >> hg_shift), tokens - 1), pv.max_rows - 1);
        // Query row r of the tile is row row0 + from_row0(r) of q and out (the last
        // token's for rows past the `left` tokens): a 64-bit base a tile and 32 bits from
        // there.
        const int left = uniform(tokens - wk.j * tm);
        const long row0 = uniform((long)(uniform(b.off[wk.i]) + wk.j * tm) * nh + (wk.y << hg_shift));
        const char* const q_tile = (const char*)uniform(q_gate + row0 * 2 * kHd);
        char* const out_tile = (char*)uniform(out + row0 * kHd);
        auto from_row0 = [&](int r) { return min(r >> hg_shift, left - 1) * nh + (r & (hg - 1)); };

        // A wave brings 8 rows of a step's K and V; it holds 64 entries of the page
        // table, one a lane, from entry `held` on.
        int held = 0, ids = 0;
        auto hold = [&](int entry) {
            held = entry;
            ids = page_of(table, entry + lane, pv.max_pages, pv.n_pages);
        };
        auto row8 = [&](int s) { return uniform(min(s * kStep + 8 * wave, last16 + (8 * wave & 8))); };
        const int s0 = 2 * wk.t0;
        const int steps = max(1, (min(rows, wk.t1 * kUnit) - wk.t0 * kUnit + kStep - 1) / kStep);
        hold(row8(s0) >> pv.page_shift);
        auto group_at = [&](int s) {
            const int r = row8(s), entry = r >> pv.page_shift;
            if (__builtin_expect(uniform(entry - held) >= kWave, 0)) hold(entry);
            return row_offset<float>(pv, __builtin_amdgcn_readlane(ids, uniform(entry - held)), kvh, r);
        };
        uint32_t ko[8], vo[2];
#pragma unroll
        for (int i = 0; i < 8; ++i) ko[i] = 16u * (lane ^ ((8 * wave + i) & 15));
        vo[0] = 16u * lane;
        vo[1] = 16u * (lane ^ 8);
        auto issue_k = [&](int i, const void* from, int buf) { dma_nth(i, from, ko[i], kaddr + buf * kBuf); };
        auto issue_v = [&](int i, const void* from, int buf) { dma_nth(i, from, vo[i >> 2], vaddr + buf * kBuf); };
        auto k_from = [&](size_t at) { return uniform((const float*)pv.k + at); };
        auto v_from = [&](size_t at) { return uniform((const float*)pv.v + at); };

        // q rows to where V will be, 16-byte chunks permuted by row (chunk ^ row % 32).
        const float4* const qs = reinterpret_cast<const float4*>(&st.v[0][0][0]);
#pragma unroll 4
        for (int r = 16 * wave; r < 16 * wave + 16; ++r)
            dma_nth(0, q_tile, from_row0(r) * (2 * kHd * 4) + 16 * (lane ^ (r & 31)),
                     lds_address(&st.v[0][0][0]) + r * kHd * 4);
        const size_t at0 = group_at(s0);
#pragma unroll
        for (int i = 0; i < 8; ++i) issue_k(i, k_from(at0), 0);
        size_t at1 = group_at(s0 + 1), at2 = group_at(s0 + 2);
        if (tid == 0) st.found = 0;

        // q: lane (row nn, h) has dims 128 half + 16 s + 8 h + j of its row, s < 8.
        Cut3 q[8];
        {
            float x[8][8];
            const float scale = q_row(x, qs + (32 * rg + nn) * (kHd / 4), pv.rope + (size_t)mine * kRopeDim, st.ss, rg, half,
                                      lane, eps);
            const float* const w = &st.w[128 * half + 8 * h];
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                float y[8];
#pragma unroll
                for (int c = 0; c < 8; c += 4) {
                    const float4 v = *reinterpret_cast<const float4*>(&w[16 * s + c]);
                    y[c] = x[s][c] * (scale * v.x);
                    y[c + 1] = x[s][c + 1] * (scale * v.y);
                    y[c + 2] = x[s][c + 2] * (scale * v.z);
                    y[c + 3] = x[s][c + 3] * (scale * v.w);
                }
                q[s] = cut3(y);
            }
        }

        f32x16 o[4];                                       // dims 128 half + 32 d + row at [d]
        auto pin = [&]() { asm volatile("" : "+a"(o[0]), "+a"(o[1]), "+a"(o[2]), "+a"(o[3])); };
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int k = 0; k < 16; ++k) o[d][k] = 0.0f;
        pin();
        float m_run = -INFINITY, l_run = 0.0f;

        // K: lane (row nn, h), dims 128 half + 16 s + 8 h ..; V of 16 rows and 32 dims:
        // lane (dim nn, h), rows 4 h + {0 .. 3, 8 .. 11}.
        uint32_t ka[8], va[4];
#pragma unroll
        for (int s = 0; s < 8; ++s)
            ka[s] = lds_address(&st.k[0][nn][128 * half]) + 16 * ((4 * (s >> 1) + 2 * h + (s & 1)) ^ (nn & 15));
#pragma unroll
        for (int d = 0; d < 4; ++d) va[d] = lds_address(&st.v[0][4 * h][128 * half]) + 4 * (32 * (d ^ h) + nn);
        auto k_read = [&](int s, float (&y)[8]) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const f32x4 a = *(lds_f32x4*)(uintptr_t)(ka[2 * (s & 3) + c] + 256 * (s >> 2));
#pragma unroll
                for (int k = 0; k < 4; ++k) y[4 * c + k] = a[k];
            }
        };
        auto v_read = [&](int row16, int d, float (&y)[8]) {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = *(lds_float*)(uintptr_t)(va[d] + (row16 + (j & 3) + 8 * (j >> 2)) * kHd * 4);
        };
        // The wave's half of a step's scores, to its partner; beside(s, i) behind the i-th
        // product of operand s.
        f32x16 x;
        auto scores = [&](auto beside) {
            float y[2][8];
            k_read(0, y[0]);
            k_read(1, y[1]);
#pragma unroll
            for (int k = 0; k < 16; ++k) x[k] = 0.0f;
            Cut3 a = cut3(y[0]);
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                if (s + 2 < 8) k_read(s + 2, y[s & 1]);
                Cutter c;
                x = mul6(a, q[s], x, [&](int i) {
                    if (s + 1 < 8) c.stage(y[(s + 1) & 1], i);
                    beside(s, i);
                });
                if (s + 1 < 8) a = c.done();
            }
#pragma unroll
            for (int c = 0; c < 4; ++c)
                st.x[wave][c][lane] = make_float4(x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]);
        };

#pragma unroll
        for (int i = 0; i < 8; ++i) {
            issue_v(i, v_from(at0), 0);
            issue_k(i, k_from(at1), 1);
        }
        scores([](int, int) {});
        int buf = 0;
        // What the scores say of a step: its weights, in three parts.
        Cut3 p[2];
        auto weigh = [&](int s) {
            const int base = s * kStep;
            float sc[16];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float4 y = st.x[wave ^ 2][c][lane];
                sc[4 * c] = x[4 * c] + y.x; sc[4 * c + 1] = x[4 * c + 1] + y.y;
                sc[4 * c + 2] = x[4 * c + 2] + y.z; sc[4 * c + 3] = x[4 * c + 3] + y.w;
            }
            if (base + kStep - 1 > first) {
                asm volatile("");                          // a branch, not selects
                const int lim = mine - base - 4 * h;
#pragma unroll
                for (int k = 0; k < 16; ++k) sc[k] = 8 * (k >> 2) + (k & 3) <= lim ? sc[k] : -INFINITY;
            }
            float mx = fmaxf(sc[0], sc[1]);
#pragma unroll
            for (int k = 2; k < 16; ++k) mx = fmaxf(mx, sc[k]);
            mx = xor32_max(mx);
            if (__builtin_expect_with_probability(__any(mx > m_run), 0, 0.99)) {   // (m_run is -inf at first)
                const float m_new = mx > m_run ? mx + kMove : m_run;
                const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.0f : m_new));
                m_run = m_new;
                l_run *= alpha;
                pin();
#pragma unroll
                for (int d = 0; d < 4; ++d) o[d] *= alpha;
                pin();
            }
            const float sub = m_run == -INFINITY ? 0.0f : m_run;
            float sum = 0.0f;                              // (of the step, as the fp16 kernel's of a unit)
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                sc[k] = __builtin_amdgcn_exp2f(sc[k] - sub);
                sum += sc[k];
            }
            l_run += sum;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float y[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] = sc[8 * c + k];
                p[c] = cut3(y);
            }
        };
        auto output = [&]() {
            float y[2][8];
            v_read(0, 0, y[0]);
            v_read(0, 1, y[1]);
            Cut3 a = cut3(y[0]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i + 2 < 8) v_read(16 * ((i + 2) >> 2), (i + 2) & 3, y[i & 1]);
                Cutter c;
                o[i & 3] = mul6(a, p[i >> 2], o[i & 3], [&](int k) {
                    if (i + 1 < 8) c.stage(y[(i + 1) & 1], k);
                });
                if (i + 1 < 8) a = c.done();
            }
        };
        auto guard = [&](int s) {
            if (s * kStep + kStep - 1 > first)
                guard_rows<8>(&st.v[buf][8 * wave][0], s * kStep + 8 * wave, rows, &st.found, first, lane);
        };
#pragma nounroll
        for (int s = s0; s + 1 < s0 + steps; ++s) {
            dma_wait();
            lds_barrier();                                 // rows, and the partner's scores
            guard(s);
            weigh(s);
            lds_barrier();                                 // the scores are read
            const int flip = buf ? -kBuf : kBuf;
#pragma unroll
            for (int i = 0; i < 8; ++i) ka[i] += flip;
            const void* const next_k = k_from(at2);
            const void* const next_v = v_from(at1);
            at1 = at2;
            at2 = group_at(s + 3);
            scores([&](int i, int k) {
                if (k == 2) issue_k(i, next_k, buf);
                if (k == 5) issue_v(i, next_v, buf ^ 1);
            });
            output();
#pragma unroll
            for (int d = 0; d < 4; ++d) va[d] += flip;
            buf ^= 1;
        }
        dma_wait();
        lds_barrier();
        const bool whole = wk.t0 == 0 && wk.t1 == wk.tiles;
        float4 gate[16];                                   // of the wave's rows 16 wave ..
        if (whole) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
                gate[r] = *reinterpret_cast<const float4*>(
                    q_tile + (uint32_t)(from_row0(16 * wave + r) * (2 * kHd * 4) + 4 * kHd + 16 * lane));
        }
        guard(s0 + steps - 1);
        weigh(s0 + steps - 1);
        lds_barrier();                                     // the guarded rows
        output();
        pin();

        asm volatile("" : "+v"(lane), "+v"(nn));
        const int slot = 2 * wg + (wk.t0 == 0);
        l_run = xor32_sum(l_run);
        if (lane < 32) st.ss[wave][nn] = half ? m_run : l_run;
        lds_barrier();                                     // K and V are read
        float4* const os = reinterpret_cast<float4*>(&st.k[0][0][0]);
        put_rows(os, o, rg, half, lane);
        lds_barrier();
        const int row = 16 * wave + (lane & 15);
        const float l = st.ss[row >> 5][row & 31];
        float* const to_part = part_o + (size_t)slot * kPagedTileRows * kHd;
        auto gate_row = [&](int r) { return q_tile + (uint32_t)(from_row0(r) * (2 * kHd * 4) + 4 * kHd + 16 * lane); };
        auto out_row = [&](int r) { return r >> hg_shift < left ? out_tile + (uint32_t)(from_row0(r) * (kHd * 4) + 16 * lane) : nullptr; };
        const bool look = leave_rows(os, l, st.ss[2 + (row >> 5)][row & 31], whole, gate, to_part,
                                     part_ml + (size_t)2 * slot * kPagedTileRows, wave, lane, out_row);
        if (__builtin_expect(look || uniform(st.found), 0))
            settle_rows<float>(os, pv, table, kvh, wk.t0 * kUnit, min(rows, wk.t1 * kUnit), first, left, hg_shift, l, whole,
                            to_part, wave, lane, gate_row, out_row);
        lds_barrier();                                     // (the stores need no wait)
    }
}

// ---- joining cut tiles ------------------------------------------------------

// 16 query rows of one tile a workgroup, where the tile's units went to several
// workgroups: four rows a wave together, a lane four dims.  Bound by latency: four
// rows' parts are asked for four at a time, their maxima and sums 16 at a time, a
// lane each (row lane / 16).  13 parts of 36 tiles: 7 us (one row after the other,
// 15).
__global__ __launch_bounds__(NT) void paged_prefill_merge(PagedView pv, PagedBatch b, const float* __restrict__ part_o,
                                                          const float* __restrict__ part_ml,
                                                          const float* __restrict__ q_gate, float* __restrict__ out,
                                                          int hg_shift, int ng, int nwg) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int groups = pv.nkv * ng, nh = groups << hg_shift, tm = kPagedTileRows >> hg_shift;
    const Units un = units_of(pv, b, groups, hg_shift, 0, lane);
    const long per = (un.total + nwg - 1) / nwg;
    // The workgroup's tile: the sequences' tiles in order.
    int tile_end = lane < b.n ? ((b.off[lane + 1] - b.off[lane] + tm - 1) / tm) * groups : 0;
    for (int o = 1; o < b.n; o <<= 1) {
        const int x = __shfl_up(tile_end, o, kWave);
        if (lane >= o) tile_end += x;
    }
    const int q = blockIdx.x >> 2;
    const int i = __popcll(__ballot(lane < b.n && tile_end <= q));
    const int tokens = b.off[i + 1] - b.off[i];
    const Tiles ts(__builtin_amdgcn_readlane(un.start, i), tokens, hg_shift, un.more);
    const int local = q - (__builtin_amdgcn_readlane(tile_end, i) - ts.n * groups);
    const int y = local / ts.n, o = local - y * ts.n, j = ts.tile(o);
    const long each = ts.before(ts.n);
    const long s = readlane_long(un.end, i) - each * groups + y * each + ts.ordered(o);
    const int w0 = (int)(s / per), w1 = (int)((s + ts.cnt(j) - 1) / per);
    if (w0 == w1) return;
    const int row0 = (blockIdx.x & 3) * 16 + 4 * wave;
    auto token = [&](int r) { return j * tm + ((row0 + r) >> hg_shift); };
    auto row_of = [&](int r) {
        return (size_t)(b.off[i] + min(token(r), tokens - 1)) * nh + (y << hg_shift) + ((row0 + r) & ((1 << hg_shift) - 1));
    };
    // Part of workgroup w: its last segment for the first one, else its first.
    auto part = [&](int w, int r) { return (size_t)(2 * w + (w == w0)) * kPagedTileRows + row0 + r; };
    const int mine = lane >> 4, at = lane & 15;
    float4 gate[4], x[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        gate[r] = *reinterpret_cast<const float4*>(q_gate + row_of(r) * 2 * kHd + kHd + 4 * lane);
        x[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float M = -INFINITY, l = 0.0f;
    for (int w = w0 + at; w <= w1; w += 16) M = fmaxf(M, part_ml[2 * part(w, mine)]);
    M = row_max(M);
    const float mu = M == -INFINITY ? 0.0f : M;
    for (int c = w0; c <= w1; c += 16) {
        float f = 0.0f;                                    // of part c + at
        if (c + at <= w1) {
            // a part none of whose rows this row sees has maximum -inf
            const float2 ml = *reinterpret_cast<const float2*>(part_ml + 2 * part(c + at, mine));
            f = __builtin_amdgcn_exp2f(ml.x - mu);
            l += f * ml.y;
        }
        constexpr int U = 4;
        for (int w = c; w <= min(w1, c + 15); w += U) {
            float4 p[4][U];
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int k = 0; k < U; ++k) p[r][k] = reinterpret_cast<const float4*>(part_o + part(min(w + k, w1), r) * kHd)[lane];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                if (w + k > w1) break;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float g = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), 16 * r + w + k - c));
                    x[r].x += g * p[r][k].x; x[r].y += g * p[r][k].y; x[r].z += g * p[r][k].z; x[r].w += g * p[r][k].w;
                }
            }
        }
    }
    const float inv_l = 1.0f / row_sum(l);
    if (__builtin_expect(__any(not_finite(x[0]) || not_finite(x[1]) || not_finite(x[2]) || not_finite(x[3])), 0)) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {                      // an infinity outlasts a weight of 0
            const float top = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, mu), 16 * r));
            x[r] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma nounroll
            for (int w = w0; w <= w1; ++w)
                x[r] = plus_weighted(x[r], __builtin_amdgcn_exp2f(part_ml[2 * part(w, r)] - top),
                                     reinterpret_cast<const float4*>(part_o + part(w, r) * kHd)[lane]);
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const float inv = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, inv_l), 16 * r));
        x[r] = gated(make_float4(x[r].x * inv, x[r].y * inv, x[r].z * inv, x[r].w * inv), gate[r]);
        if (token(r) < tokens) *reinterpret_cast<float4*>(out + row_of(r) * kHd + 4 * lane) = x[r];
    }
}

int prefill_workgroups(const q35m_ctx* c) { return c->n_cu; }

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
    long longest = 0;                                      // rows that a tile may see
    for (int i = 0; i < b.n; ++i) {
        const long n = ((long)b.off[i + 1] - b.off[i] + tm - 1) / tm;
        tiles += n * c->d.nkv * ng;
        if (n) longest = std::max(longest, p->map.length(b.seq[i]) + n * tm);
    }
    // Short tiles that each get a workgroup are not cut, and nothing is to be joined,
    // as the lengths known here say (not so those of a replay): up to 4 units of an
    // fp16 cache (30 tokens: 8.6 us against 11.0 with the joining; 230: 14.5 against
    // 15.5), up to 2 of an fp32 one (13.7 against 15.4 for four sequences of 120 rows;
    // 4 units are slower, 21 against 18).
    const int shift = p->type == Q35M_KV_F16 ? 2 : 1;
    const int more = tiles <= nwg && longest <= kUnit << shift && !p->capturing() ? shift : 0;
    {
        ProfScope ps(c, K_PAGED_PREFILL);
        auto go = [&](auto kern) {
            hipExtLaunchKernelGGL(kern, dim3(nwg), dim3(NT), 0, c->stream, ps.a, ps.b, 0, pv, b, q_gate, L.q_norm, out,
                                  part_o, part_ml, hg_shift, ng, more, c->d.eps);
        };
        if (p->type == Q35M_KV_F16) go(paged_prefill_f16);
        else go(paged_prefill_f32);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (more) return hipSuccess;
    ProfScope ps(c, K_PAGED_PREFILL_MERGE);
    hipExtLaunchKernelGGL(paged_prefill_merge, dim3((unsigned)(4 * tiles)), dim3(NT), 0, c->stream, ps.a, ps.b, 0, pv, b,
                          part_o, part_ml, q_gate, out, hg_shift, ng, nwg);
    return hipGetLastError();
}

}  // namespace q35
