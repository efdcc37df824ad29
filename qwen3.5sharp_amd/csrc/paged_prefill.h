// What the paged prefill kernels share (paged_prefill.hip says how a call's work is
// divided): a workgroup's walk over its units, loads to LDS, and the beginning and
// the end of a segment.
#pragma once

#include "paged_device.h"

namespace q35 {

// The kernel of a cache in 4 bits (paged_prefill_mx4.hip), launched as the others.
using PagedPrefillKernel = void (*)(PagedView, PagedBatch, const float*, const float*, float*, float*, float*, int, int, int,
                                    float);
PagedPrefillKernel paged_prefill_mx4_kernel();

namespace {

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
    __host__ __device__ __forceinline__ Tiles(int start, int tokens, int hg_shift, int more) : shift(hg_shift + more) {
        const int tm_shift = 6 - hg_shift, tm = 1 << tm_shift;
        n = (tokens + tm - 1) >> tm_shift;
        q0 = ((long)start + tm + (kUnit << more) - 1) >> tm_shift;
    }
    __host__ __device__ __forceinline__ long floors(long m) const {      // sum of floor(y / hg) over y < m
        const long k = m >> shift;
        return ((k * (k - 1)) >> 1 << shift) + k * (m - (k << shift));
    }
    __host__ __device__ __forceinline__ long cnt(int j) const { return (q0 + j) >> shift; }
    __host__ __device__ __forceinline__ long before(int j) const { return floors(q0 + j) - floors(q0); }   // tiles < j
    // Units of tiles j and n - 1 - j together, if all of them are in pairs of as many (else 0): two
    // numbers whose sum is hg - 1 modulo hg have remainders that add up to hg - 1.
    __host__ __device__ __forceinline__ long pair() const {
        const long sum = 2 * q0 + n - 1, last = (1L << shift) - 1;
        return n % 2 == 0 && (sum & last) == last ? (sum - last) >> shift : 0;
    }
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

// In 4 bits tiles are left whole, dealt out in pairs of first and last, which are alike,
// where that leaves the busiest workgroup up to 12 units more than cutting: a cut tile
// is begun and ended once more, 14 us at 1.5 a unit, and joined.  1000 tokens, 16 units
// for 9: 46 us against 66; 2000, 34 for 32: 91 against 111; 800 behind 1000, 29 for 18: 66.5
// against 69.5; 512 behind 1000, 24 for 11: 58.5 against 54.
// Returned is log2 of what a unit is over 64 rows then, of which a tile has one (0: cut).
// longest: rows that a tile may see; pair: units of a sequence's first and last tile.
__host__ __device__ __forceinline__ int whole_tiles(long tiles, long units, int longest, int pair, int nwg) {
    const unsigned rounds = (unsigned)((unsigned)tiles + nwg - 1) / (unsigned)nwg;
    const long most = (long)(rounds >> 1) * (pair + 1) + (rounds & 1) * ((longest + kUnit - 1) / kUnit);
    if ((most - 12) * nwg > units) return 0;
    const unsigned more = (unsigned)(longest - 1) / kUnit;
    return more < 2 ? 1 : 32 - __builtin_clz(more);
}
__device__ __forceinline__ Units units_or_whole(const PagedView& pv, const PagedBatch& b, int groups, int hg_shift, int nwg,
                                                int lane) {
    Units u;
    u.start = 0;
    u.end = 0;
    int tiles = 0, longest = 1, pair = 0;                  // (the last two: of this and the sequences before)
    const int tokens = lane < b.n ? b.off[lane + 1] - b.off[lane] : 0;
    if (lane < b.n) u.start = pv.lens[b.seq[lane]];
    if (tokens) {
        const Tiles t(u.start, tokens, hg_shift, 0);
        u.end = t.before(t.n) * groups;
        tiles = t.n * groups;
        longest = u.start + (t.n << (6 - hg_shift));
        pair = (int)(t.cnt(0) + t.cnt(t.n - 1));
    }
    for (int o = 1; o < b.n; o <<= 1) {
        const long x = shfl_up_long(u.end, o);
        const int y = __shfl_up(tiles, o, kWave), z = __shfl_up(longest, o, kWave), p = __shfl_up(pair, o, kWave);
        if (lane >= o) {
            u.end += x;
            tiles += y;
            longest = max(longest, z);
            pair = max(pair, p);
        }
    }
    auto all = [&](int v) { return __builtin_amdgcn_readlane(v, b.n - 1); };
    u.total = readlane_long(u.end, b.n - 1);
    u.more = whole_tiles(all(tiles), u.total, all(longest), all(pair), nwg);
    if (u.more) {
        u.end = tiles;
        u.total = all(tiles);
    }
    if (lane >= b.n) u.end = u.total;
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
// lane's place (none if null), or as parts.  gate_of(k): the gate of the wave's k-th row, if whole.  l, m: sum and maximum of row 16 wave + lane % 16.
// Whether a value of theirs is not finite.
template <typename G, typename F>
__device__ __forceinline__ bool leave_rows(const float4* os, float l, float m, bool whole, G gate_of, float* part_o,
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
        float4 gate[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            gate[k] = gate_sigmoid(gate_of(k));
            asm volatile("" : "+v"(gate[k].x), "+v"(gate[k].y), "+v"(gate[k].z), "+v"(gate[k].w));
        }
        auto put = [&](int k, float4 x) {
            const float inv = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, inv_l), k));
            const float4 g = gate[k];
            x = make_float4(x.x * inv * g.x, x.y * inv * g.y, x.z * inv * g.z, x.w * inv * g.w);
            if (char* to = out_row(16 * wave + k)) to_global(to, x);
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

}  // namespace
}  // namespace q35
