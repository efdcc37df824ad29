// Paged K/V cache: attention of one new token per sequence.
//
// Per sequence at length p, q head h of kv head g: q = norm(rope(q, p)) (1 + w),
// s_j = q . K_j / 16 over rows j = 0 .. p (the p cached rows and the new one),
// out = sigmoid(gate) sum_j e^{s_j - m} V_j / sum_j e^{s_j - m}: DecodeAttention
// after the projections (src/Qwen35Sharp.Model/Qwen35Model.Decode.cs:294-323).
// Every cached row is read once, so the bound is the cache's bytes over HBM's
// rate; the products are a few operations a byte.
//
// Work is cut into units of 64 (fp32) or 128 (fp16) rows of one (sequence, head
// group) and dealt out evenly: workgroup w takes units [w per, (w + 1) per) of the units of all
// sequences in order, per = ceil(units / workgroups), both found on the device
// from the lengths there, so batches of unequal lengths fill the card and a
// captured launch fits any lengths.  A stretch of units of one (sequence, head
// group) is a segment: whole ones are finished where they are, of the others
// the maximum, the sum and the unnormalised output go to the workspace (two
// segments of a workgroup at most are not whole, its first and its last), and
// paged_decode_merge joins them.  (Larger units where no sequence has to be cut:
// launch_paged_decode.)
//
// A unit's rows go to the four waves, which keep an online softmax each and
// meet at the segment's end.  All products are matrix instructions with the
// (up to 16) q heads of the kv head as columns:
//   S^T = K Q^T  (rows of K: the 16 lanes l % 16; dims: lane group l / 16)
//   O^T = V^T P^T, whose P^T operand is S^T's own register layout (a lane
//   holds, of its q column, rows 4 (l / 16) + i), with V rows read in that
//   order; so neither P nor V crosses lanes.
// fp32 caches use the fp32 instruction (16 x 16 x 4).  fp16 caches use
// 16 x 16 x 32 on fp16 with the fp32 operands q and P as two fp16 values each
// (hi + lo, to 2^-23 of the value; q's row and P scaled by powers of two into the range),
// and a register transpose of V (8 rows x 8 dims a lane).
// The waves share the forming of q rows through LDS: formed in every wave, behind
// K and V in the queue of loads, they cost a call over 8192 rows 2 of its 13 us
// (now 9.4, of which the 33.5 MB take 4.9 and two launches the most of the rest).
// Two tiles a wave in flight instead of one spill, and K's alone are no faster.
#include "paged_device.h"

namespace q35 {
namespace {

constexpr int NT = 256;
constexpr float kLog2e = 1.4426950408889634f;
// P is formed as e^{s - m} 2^kPShift (the normalisation divides the factor out).  fp16:
// the largest weight is at the upper end of the range, so that the steps of a weight's
// low half, 2^-24, are 2^-39 of it.  fp32: weights up to one, so that an output overflows
// only where the sum of |V| over the rows does.
template <typename T>
constexpr float kPShift = std::is_same_v<T, float> ? 0.0f : 15.0f;

// How a wave reads K.  The operand's own shape, 16 rows x 64 bytes an instruction,
// takes half a cache line of a row at a time, which reads slower than whole lines:
// 120 us against 112 for 64 sequences of up to 4000 fp16 rows (709 MB, 6.3 TB/s),
// 247 against 220 for 8 of up to 32768 fp32 rows (1.52 GB, 6.9 TB/s).  (Whole lines
// and an exchange between lanes l and l ^ 8 in front of the products: 128 and 261.)
// So up to 8 q heads (S) it is 8 rows x 128 bytes: a lane has row l % 8 and 16-byte
// chunk 2 g + l / 8 % 2 of the line, g = l / 16.  As an operand these are 16 rows of which the
// upper 8 are the lower ones' odd chunks; q's columns are as well: column n < 8 is
// head n's even chunks, column n + 8 its odd ones.  The product's quarter (lower
// rows, lower columns) is the even chunks' part of a score and the quarter (upper,
// upper) the odd ones'; the rest is not used.  joined() adds the two, of a product
// of rows 0 .. 7 and one of rows 8 .. 15: to lane (n, g) rows 4 g + i.
__device__ __forceinline__ float joined(float a, float b) {
    const auto x = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), false, false);
    return __builtin_bit_cast(float, (uint32_t)x[0]) + row_xor<8>(__builtin_bit_cast(float, (uint32_t)x[1]));
}

template <typename T, bool S>
struct Tile;

// 16 rows of an fp32 cache a wave.
template <bool S>
struct Tile<float, S> {
    static constexpr int kRows = 16;
    float q[S ? 32 : 64];   // dims 16 t + 4 g + c at [4 t + c]; S: 32 t + 8 g + 4 (l / 8 % 2) + c
    float4 k[16], v[4][4];  // K row l % 16, dims 16 t + 4 g (S: see above, rows 0 .. 7 at [2 t]); V row 4 g + i, dims 64 t + 4 m
    f32x4 o[16];            // dims 64 t + 4 row + c at [4 t + c]

    // q row n in LDS, 16-byte chunks permuted: chunk ^ n.
    static __device__ __forceinline__ void put_q(float4* row, int r, float4 x, int lane) { row[lane ^ r] = x; }
    __device__ __forceinline__ void load_q(const float4* row, int n, int lane) {
        const int g = lane >> 4, odd = (lane >> 3) & 1;
#pragma unroll
        for (int t = 0; t < (S ? 8 : 16); ++t) {
            const float4 a = row[(S ? 8 * t + 2 * g + odd : 4 * t + g) ^ n];
            q[4 * t] = a.x; q[4 * t + 1] = a.y; q[4 * t + 2] = a.z; q[4 * t + 3] = a.w;
        }
    }

    __device__ __forceinline__ void load_k(const float* p, int, int lane) {
        const float* a = p + (lane & (S ? 7 : 15)) * kHd + 4 * (lane >> (S ? 3 : 4));
#pragma unroll
        for (int t = 0; t < 16; ++t) k[t] = load_nt(a + (S ? 32 * (t >> 1) + 8 * (t & 1) * kHd : 16 * t));
    }
    __device__ __forceinline__ void load_v(const float* p, int, int lane) {
        const float* a = p + (lane >> 4) * 4 * kHd + 4 * (lane & 15);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int t = 0; t < 4; ++t) v[i][t] = load_nt(a + i * kHd + 64 * t);
    }
    // Row `at` of the tile (none if negative) comes from kn / vn, rows from
    // `rows` on are masked: their V must not meet the products (0 x NaN).
    __device__ __forceinline__ void fix(const float* kn, const float* vn, int at, int rows, int lane) {
        const int g = lane >> 4, m = lane & 15;
#pragma unroll
        for (int t = 0; t < 16; ++t)
            if (S) {
                if ((m & 7) + 8 * (t & 1) == at) k[t] = *reinterpret_cast<const float4*>(kn + 32 * (t >> 1) + 4 * (lane >> 3));
            } else if (m == at) {
                k[t] = *reinterpret_cast<const float4*>(kn + 16 * t + 4 * g);
            }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if (4 * g + i == at) v[i][t] = *reinterpret_cast<const float4*>(vn + 64 * t + 4 * m);
                if (4 * g + i >= rows) v[i][t] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
    }
    __device__ __forceinline__ void scores(float (&s)[4]) const {
        f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
        if constexpr (S) {
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                a = __builtin_amdgcn_mfma_f32_16x16x4f32(k[2 * t].x, q[4 * t], a, 0, 0, 0);
                b = __builtin_amdgcn_mfma_f32_16x16x4f32(k[2 * t + 1].x, q[4 * t], b, 0, 0, 0);
                a = __builtin_amdgcn_mfma_f32_16x16x4f32(k[2 * t].y, q[4 * t + 1], a, 0, 0, 0);
                b = __builtin_amdgcn_mfma_f32_16x16x4f32(k[2 * t + 1].y, q[4 * t + 1], b, 0, 0, 0);
                a = __builtin_amdgcn_mfma_f32_16x16x4f32(k[2 * t].z, q[4 * t + 2], a, 0, 0, 0);
                b = __builtin_amdgcn_mfma_f32_16x16x4f32(k[2 * t + 1].z, q[4 * t + 2], b, 0, 0, 0);
                a = __builtin_amdgcn_mfma_f32_16x16x4f32(k[2 * t].w, q[4 * t + 3], a, 0, 0, 0);
                b = __builtin_amdgcn_mfma_f32_16x16x4f32(k[2 * t + 1].w, q[4 * t + 3], b, 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int t = 0; t < 16; ++t) {
                a = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t].x, q[4 * t], a, 0, 0, 0);
                b = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t].y, q[4 * t + 1], b, 0, 0, 0);
                a = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t].z, q[4 * t + 2], a, 0, 0, 0);
                b = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t].w, q[4 * t + 3], b, 0, 0, 0);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = S ? joined(a[i], b[i]) : a[i] + b[i];
    }
    static __device__ __forceinline__ int row_of(int i, int g) { return 4 * g + i; }
    static constexpr int kScores = 4;
    __device__ __forceinline__ void pv(const float (&p)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                o[4 * t] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][t].x, p[i], o[4 * t], 0, 0, 0);
                o[4 * t + 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][t].y, p[i], o[4 * t + 1], 0, 0, 0);
                o[4 * t + 2] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][t].z, p[i], o[4 * t + 2], 0, 0, 0);
                o[4 * t + 3] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][t].w, p[i], o[4 * t + 3], 0, 0, 0);
            }
    }
    // The lane's output values, 4 consecutive dims at a time.
    template <typename F>
    __device__ __forceinline__ void each4(int g, F f) const {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                f(64 * t + 4 * (4 * g + i), make_float4(o[4 * t][i], o[4 * t + 1][i], o[4 * t + 2][i], o[4 * t + 3][i]));
    }
};

// 32 rows of an fp16 cache a wave, as two groups of 16.
template <bool S>
struct Tile<_Float16, S> {
    static constexpr int kRows = 32;
    f16x8 qh[S ? 4 : 8], ql[S ? 4 : 8];        // dims 32 t + 8 g ..; S: 64 t + 16 g + 8 (l / 8 % 2) ..
    u32x4 k[2][8], v[2][8];    // K row l % 16 of group kb, dims 32 t + 8 g (S: as above); V row 16 (j / 4) + 4 g + j % 4, dims 128 u + 8 m
    f32x4 o[16];               // dims 128 u + 8 row + b at [8 u + b]

    // The row, already scaled into fp16's range, as hi (chunks 0 .. 31) and lo.
    static __device__ __forceinline__ void put_q(float4* row, int r, float4 x, int lane) {
        f16x2 h[2], l[2];
        split16(x.x, x.y, h[0], l[0]);
        split16(x.z, x.w, h[1], l[1]);
        f16x2* const at = reinterpret_cast<f16x2*>(row + ((lane >> 1) ^ r)) + 2 * (lane & 1);
        at[0] = h[0]; at[1] = h[1];
        f16x2* const to = reinterpret_cast<f16x2*>(row + (32 + (lane >> 1) ^ r)) + 2 * (lane & 1);
        to[0] = l[0]; to[1] = l[1];
    }
    __device__ __forceinline__ void load_q(const float4* row, int n, int lane) {
        const int g = lane >> 4, odd = (lane >> 3) & 1;
#pragma unroll
        for (int t = 0; t < (S ? 4 : 8); ++t) {
            const int at = S ? 8 * t + 2 * g + odd : 4 * t + g;
            qh[t] = __builtin_bit_cast(f16x8, row[at ^ n]);
            ql[t] = __builtin_bit_cast(f16x8, row[(32 + at) ^ n]);
        }
    }

    __device__ __forceinline__ void load_k(const _Float16* p, int kb, int lane) {
        const _Float16* a = p + (lane & (S ? 7 : 15)) * kHd + 8 * (lane >> (S ? 3 : 4));
#pragma unroll
        for (int t = 0; t < 8; ++t)
            k[kb][t] = __builtin_nontemporal_load(
                reinterpret_cast<const u32x4*>(a + (S ? 64 * (t >> 1) + 8 * (t & 1) * kHd : 32 * t)));
    }
    __device__ __forceinline__ void load_v(const _Float16* p, int kb, int lane) {
        const _Float16* a = p + (lane >> 4) * 4 * kHd + 8 * (lane & 15);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u)
                v[u][4 * kb + i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a + i * kHd + 128 * u));
    }
    __device__ __forceinline__ void fix(const _Float16* kn, const _Float16* vn, int at, int rows, int lane) {
        const int g = lane >> 4, m = lane & 15;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int t = 0; t < 8; ++t)
                if (S) {
                    if (16 * kb + (m & 7) + 8 * (t & 1) == at)
                        k[kb][t] = *reinterpret_cast<const u32x4*>(kn + 64 * (t >> 1) + 8 * (lane >> 3));
                } else if (16 * kb + m == at) {
                    k[kb][t] = *reinterpret_cast<const u32x4*>(kn + 32 * t + 8 * g);
                }
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int r = row_of(j, g);
                if (r == at) v[u][j] = *reinterpret_cast<const u32x4*>(vn + 128 * u + 8 * m);
                if (r >= rows) v[u][j] = u32x4{0, 0, 0, 0};
            }
    }
    __device__ __forceinline__ void scores(float (&s)[8]) const {
        if constexpr (S) {
            f32x4 a[4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
            // 8 rows each; the low halves' products first
            auto all = [&](const f16x8 (&q)[4]) {
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        a[r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, k[r >> 1][2 * t + (r & 1)]), q[t], a[r], 0, 0, 0);
            };
            all(ql);
            all(qh);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[i] = joined(a[0][i], a[1][i]);
                s[4 + i] = joined(a[2][i], a[3][i]);
            }
        } else {
            f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
            auto all = [&](const f16x8 (&q)[8]) {
#pragma unroll
                for (int t = 0; t < 8; ++t) {
                    a = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, k[0][t]), q[t], a, 0, 0, 0);
                    b = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, k[1][t]), q[t], b, 0, 0, 0);
                }
            };
            all(ql);
            all(qh);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[i] = a[i];
                s[4 + i] = b[i];
            }
        }
    }
    static __device__ __forceinline__ int row_of(int j, int g) { return 16 * (j >> 2) + 4 * g + (j & 3); }
    static constexpr int kScores = 8;
    __device__ __forceinline__ void pv(const float (&p)[8]) {
        f16x8 ph, pl;
        split16(p, ph, pl);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int b = 0; b < 8; ++b) {
                // dim 128 u + 8 m + b of the lane's 8 rows
                const uint32_t sel = (b & 1) ? 0x07060302u : 0x05040100u;
                u32x4 a;
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    a[w] = __builtin_amdgcn_perm(v[u][2 * w + 1][b >> 1], v[u][2 * w][b >> 1], sel);
                const f16x8 av = __builtin_bit_cast(f16x8, a);
                o[8 * u + b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, pl, o[8 * u + b], 0, 0, 0);
                o[8 * u + b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, ph, o[8 * u + b], 0, 0, 0);
            }
    }
    template <typename F>
    __device__ __forceinline__ void each4(int g, F f) const {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int b = 0; b < 8; b += 4)
                    f(128 * u + 8 * (4 * g + i) + b,
                      make_float4(o[8 * u + b][i], o[8 * u + b + 1][i], o[8 * u + b + 2][i], o[8 * u + b + 3][i]));
    }
};

// Rows of a unit.
template <typename T>
constexpr int kUnitRows = 4 * Tile<T, true>::kRows;

// The units of a call's sequences, one sequence a lane: `end` is the number of
// units up to and with the lane's.
struct Units {
    int rows, tiles, end, total;
};
__device__ __forceinline__ Units units_of(const PagedView& pv, const PagedBatch& b, int groups, int unit, int lane) {
    Units u;
    // (the row past max_rows of a replayed call that its caller let run over)
    u.rows = lane < b.n ? min(pv.lens[b.seq[lane]] + 1, pv.max_rows) : 0;
    u.tiles = (u.rows + unit - 1) / unit;
    u.end = u.tiles * groups;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int x = __shfl_up(u.end, o, kWave);
        if (lane >= o) u.end += x;
    }
    u.total = __builtin_amdgcn_readlane(u.end, kWave - 1);
    return u;
}

template <typename T, bool S>
__global__ __launch_bounds__(NT, 1) void paged_decode(PagedView pv, PagedBatch b, const float* __restrict__ q_gate,
                                                      const float* __restrict__ knew, const float* __restrict__ vnew,
                                                      const float* __restrict__ q_norm,
                                                      const float* __restrict__ k_norm, float* __restrict__ out,
                                                      float* __restrict__ part_o, float* __restrict__ part_ml, int hg,
                                                      int ng, int unit, float eps) {
    using Tl = Tile<T, S>;
    constexpr int R = Tl::kRows;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int groups = pv.nkv * ng, nh = groups * hg;

    __shared__ __align__(16) float obuf[4][kPagedDecodeHeads][kHd];
    __shared__ float ml[4][kPagedDecodeHeads][2];
    __shared__ __align__(16) T newrow[4][2][kHd];
    __shared__ float4 qbuf[kPagedDecodeHeads][kHd / 4];

    float4 qw = *reinterpret_cast<const float4*>(q_norm + 4 * lane);
    const float4 kw = *reinterpret_cast<const float4*>(k_norm + 4 * lane);
    qw = make_float4(1.0f + qw.x, 1.0f + qw.y, 1.0f + qw.z, 1.0f + qw.w);
    const int qe = std::is_same_v<T, float> ? 0 : q_exponent(q_norm, lane);
    const float up = ldexpf(1.0f, qe), down = ldexpf(1.0f, -qe);
    const Units un = units_of(pv, b, groups, unit, lane);
    const int per = (un.total + (int)gridDim.x - 1) / (int)gridDim.x;
    int u = blockIdx.x * per;
    const int u_end = min(u + per, un.total);

    while (u < u_end) {
        const int i = __popcll(__ballot(un.end <= u));            // the unit's sequence in the batch
        const int tiles = __builtin_amdgcn_readlane(un.tiles, i);
        const int rows = __builtin_amdgcn_readlane(un.rows, i);
        const int local = u - (__builtin_amdgcn_readlane(un.end, i) - tiles * groups);
        const int y = local / tiles, t0 = local - y * tiles;      // head group, first unit of the segment
        const int t1 = min(tiles, t0 + (u_end - u));
        u += t1 - t0;
        const int kvh = y / ng, seq = b.seq[i], pos = rows - 1;
        const int* table = pv.table + (size_t)seq * pv.max_pages;
        const int first = t0 * unit + wave * R, stop = min(rows, t1 * unit);
        const int last16 = pos & ~15;

        Tl tl;
#pragma unroll
        for (int x = 0; x < 16; ++x) tl.o[x] = f32x4{0.f, 0.f, 0.f, 0.f};
        auto page16 = [&](int r) {     // page of the 16-row group at r (the last one past the end)
            return page_of(table, min(r, last16) >> pv.page_shift, pv.max_pages, pv.n_pages);
        };
        int pg[R / 16];
        auto pages = [&](int base) {
#pragma unroll
            for (int kb = 0; kb < R / 16; ++kb) pg[kb] = page16(base + 16 * kb);
        };
        auto load_k = [&](int base, const int (&p)[R / 16]) {
#pragma unroll
            for (int kb = 0; kb < R / 16; ++kb)
                tl.load_k((const T*)pv.k + row_offset<T>(pv, p[kb], kvh, min(base + 16 * kb, last16)), kb, lane);
        };
        auto load_v = [&](int base, const int (&p)[R / 16]) {
#pragma unroll
            for (int kb = 0; kb < R / 16; ++kb)
                tl.load_v((const T*)pv.v + row_offset<T>(pv, p[kb], kvh, min(base + 16 * kb, last16)), kb, lane);
        };
        // What q's rows and the new row are made of is asked for before K and V, so
        // that they are formed while those are on their way; a wave forms every
        // fourth q row, for all.
        const bool has_new = first <= pos / R * R && pos / R * R < stop && (pos / R * R - first) % (4 * R) == 0;
        if (first < stop) pages(first);
        float4 xq[kPagedDecodeHeads / 4], xk{}, xv{};
        const float* const q_rows = q_gate + ((size_t)i * nh + y * hg) * 2 * kHd + 4 * lane;
#pragma unroll
        for (int k = 0; k < kPagedDecodeHeads / 4; ++k)
            if (wave + 4 * k < hg) xq[k] = *reinterpret_cast<const float4*>(q_rows + (size_t)(wave + 4 * k) * 2 * kHd);
        if (has_new) {
            const size_t at = ((size_t)i * pv.nkv + kvh) * kHd + 4 * lane;
            xk = *reinterpret_cast<const float4*>(knew + at);
            xv = *reinterpret_cast<const float4*>(vnew + at);
        }
        double cs[4], sn[4];                     // the rotation of dims 4 (lane % 8) ..
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            cs[k] = pv.rope[(size_t)pos * kRopeDim + 4 * (lane & 7) + k];
            sn[k] = pv.rope[(size_t)pos * kRopeDim + kRopeHalf + 4 * (lane & 7) + k];
        }
        __builtin_amdgcn_sched_barrier(0);
        if (first < stop) {
            load_k(first, pg);
            load_v(first, pg);
        }
        __builtin_amdgcn_sched_barrier(0);

        // q: the rotation, the norm, the scale 1/16 (and log2 e, for exp2; and a
        // power of two for fp16).
#pragma unroll
        for (int k = 0; k < kPagedDecodeHeads / 4; ++k) {
            const int r = wave + 4 * k;
            if (r >= hg) break;
            float x[4] = {xq[k].x, xq[k].y, xq[k].z, xq[k].w}, ss = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float a = x[c], z = row_xor<8>(a), co = (float)cs[c], si = (float)sn[c];
                x[c] = lane < 8 ? a * co - z * si : lane < 16 ? z * si + a * co : a;
                ss += x[c] * x[c];
            }
            const float scale = up * (kLog2e / 16.0f) / sqrtf(wave_sum(ss) / (float)kHd + eps);
            Tl::put_q(qbuf[r], r,
                      make_float4(x[0] * (scale * qw.x), x[1] * (scale * qw.y), x[2] * (scale * qw.z), x[3] * (scale * qw.w)),
                      lane);
        }
        // The wave that holds the new row makes it (every head group needs it;
        // one writes it to the page, and none reads it from there).
        if (has_new) {
            const float4 yk = paged_key_row(xk, cs, sn, kw, lane, (double)eps);
            store_row4(&newrow[wave][0][4 * lane], yk);
            store_row4(&newrow[wave][1][4 * lane], xv);
            const int pnew = page_of(table, pos >> pv.page_shift, pv.max_pages, pv.n_pages);
            if (y % ng == 0 && pnew >= 0 && pv.lens[seq] < pv.max_rows) {
                const size_t to = row_offset<T>(pv, pnew, kvh, pos) + 4 * lane;
                store_row4((T*)pv.k + to, yk);
                store_row4((T*)pv.v + to, xv);
            }
        }
        lds_barrier();
        {
            const int r = min(S ? n & 7 : n, hg - 1);      // columns from hg on are never read
            tl.load_q(qbuf[r], r, lane);
        }

        float m_run = -INFINITY, l_run = 0.0f;
        for (int base = first; base < stop; base += 4 * R) {
            const int next = base + 4 * R;
            const bool more = next < stop;
            if (more) pages(next);
            if (base + R > pos) tl.fix(newrow[wave][0], newrow[wave][1], pos - base, rows - base, lane);
            float s[Tl::kScores];
            tl.scores(s);
            if (more) load_k(next, pg);
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < Tl::kScores; ++j) {
                s[j] = base + Tl::row_of(j, g) < rows ? s[j] * down : -INFINITY;
                mx = fmaxf(mx, s[j]);
            }
            mx = fmaxf(m_run, xor16_max(xor32_max(mx)));
            const float mu = mx == -INFINITY ? 0.0f : mx;
            const float alpha = __builtin_amdgcn_exp2f(m_run - mu);
            m_run = mx;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < Tl::kScores; ++j) {
                s[j] = __builtin_amdgcn_exp2f(s[j] - mu + kPShift<T>);
                sum += s[j];
            }
            l_run = l_run * alpha + sum;
#pragma unroll
            for (int x = 0; x < 16; ++x) tl.o[x] *= alpha;
            tl.pv(s);
            if (more) load_v(next, pg);
        }

        // The four waves of the segment join.
        l_run = xor16_sum(xor32_sum(l_run));
        if (n < hg) {
            tl.each4(g, [&](int d, float4 x) { *reinterpret_cast<float4*>(&obuf[wave][n][d]) = x; });
            if (g == 0) {
                ml[wave][n][0] = m_run;
                ml[wave][n][1] = l_run;
            }
        }
        const bool whole = t0 == 0 && t1 == tiles;
        const int slot = 2 * blockIdx.x + (t0 == 0);
        float4 gate[kPagedDecodeHeads / 4];
#pragma unroll
        for (int k = 0; k < kPagedDecodeHeads / 4; ++k)
            if (whole && wave + 4 * k < hg)
                gate[k] = *reinterpret_cast<const float4*>(q_rows + (size_t)(wave + 4 * k) * 2 * kHd + kHd);
        lds_barrier();
        bool look = false;                                 // at an output that is not finite
        auto join = [&](int r, float4 gt, bool settle, uint32_t found) {
            float M = -INFINITY, l = 0.0f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < 4; ++w) M = fmaxf(M, ml[w][r][0]);
            const float mu = M == -INFINITY ? 0.0f : M;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float e = __builtin_amdgcn_exp2f(ml[w][r][0] - mu);
                const float4 x = *reinterpret_cast<const float4*>(&obuf[w][r][4 * lane]);
                l += e * ml[w][r][1];
                o.x += e * x.x; o.y += e * x.y; o.z += e * x.z; o.w += e * x.w;
            }
            look |= not_finite(o);
            if (settle) o = settled(o, found);
            if (whole) {
                const float inv = 1.0f / l;
                *reinterpret_cast<float4*>(out + ((size_t)i * nh + y * hg + r) * kHd + 4 * lane) =
                    gated(make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv), gt);
            } else {
                const size_t at = (size_t)slot * kPagedDecodeHeads + r;
                *reinterpret_cast<float4*>(part_o + at * kHd + 4 * lane) = o;
                if (lane == 0) *reinterpret_cast<float2*>(part_ml + 2 * at) = make_float2(M, l);
            }
        };
#pragma unroll
        for (int k = 0; k < kPagedDecodeHeads / 4; ++k) {
            if (wave + 4 * k >= hg) break;
            join(wave + 4 * k, gate[k], false, 0);
        }
        if (__builtin_expect(__any(look), 0)) {            // once more, with the infinities among the rows
            uint32_t found = infinite_rows<T>(pv, table, kvh, t0 * unit, min(stop, pos), lane);
            if (pos < stop) {                              // the new row, as the cache holds it
                const float4 x = *reinterpret_cast<const float4*>(vnew + ((size_t)i * pv.nkv + kvh) * kHd + 4 * lane);
                found |= infinite(make_float4((float)(T)x.x, (float)(T)x.y, (float)(T)x.z, (float)(T)x.w));
            }
#pragma nounroll
            for (int r = wave; r < hg; r += 4)
                join(r, *reinterpret_cast<const float4*>(q_rows + (size_t)r * 2 * kHd + kHd), true, found);
        }
        lds_barrier();
    }
}

// The parts of one (sequence, q head), where its units went to several
// workgroups: waves take parts in turn, a lane four dims.
constexpr int MW = 8;      // waves
template <typename T>
__global__ __launch_bounds__(MW * kWave) void paged_decode_merge(PagedView pv, PagedBatch b,
                                                                 const float* __restrict__ part_o,
                                                                 const float* __restrict__ part_ml,
                                                                 const float* __restrict__ q_gate,
                                                                 float* __restrict__ out, int hg, int ng, int nwg) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int groups = pv.nkv * ng, nh = groups * hg;
    const int i = blockIdx.y, head = blockIdx.x, y = head / hg, h = head - y * hg;
    const Units un = units_of(pv, b, groups, kUnitRows<T>, lane);
    const int per = (un.total + nwg - 1) / nwg;
    const int tiles = __builtin_amdgcn_readlane(un.tiles, i);
    const int s = __builtin_amdgcn_readlane(un.end, i) - tiles * groups + y * tiles;
    const int w0 = s / per, w1 = (s + tiles - 1) / per;      // its first and last workgroup
    if (w0 == w1) return;
    const size_t row = (size_t)i * nh + head;
    const float4 gate = *reinterpret_cast<const float4*>(q_gate + row * 2 * kHd + kHd + 4 * lane);
    __shared__ float4 obuf[MW][kWave];
    __shared__ float lbuf[MW];
    // Part of workgroup w: its last segment for the first one, else its first.
    auto part = [&](int w) { return (size_t)(2 * w + (w == w0)) * kPagedDecodeHeads + h; };
    float M = -INFINITY;
    for (int w = w0 + lane; w <= w1; w += kWave) M = fmaxf(M, part_ml[2 * part(w)]);
    M = wave_max(M);
    const float mu = M == -INFINITY ? 0.0f : M;
    float l = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int U = 4;       // parts whose loads are in flight together
    for (int w = w0 + wave; w <= w1; w += U * MW) {
        float4 x[U];
        float e[U], ls[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const size_t at = part(min(w + k * MW, w1));
            x[k] = reinterpret_cast<const float4*>(part_o + at * kHd)[lane];
            e[k] = part_ml[2 * at];
            ls[k] = part_ml[2 * at + 1];
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            if (w + k * MW > w1) break;
            const float f = __builtin_amdgcn_exp2f(e[k] - mu);
            l += f * ls[k];
            o.x += f * x[k].x; o.y += f * x[k].y; o.z += f * x[k].z; o.w += f * x[k].w;
        }
    }
    obuf[wave][lane] = o;
    if (lane == 0) lbuf[wave] = l;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
        for (int w = 1; w < MW; ++w) {
            const float4 x = obuf[w][lane];
            o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
            l += lbuf[w];
        }
        if (__builtin_expect(__any(not_finite(o)), 0)) {       // an infinity outlasts a weight of 0
            o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma nounroll
            for (int w = w0; w <= w1; ++w) {
                const size_t at = part(w);
                o = plus_weighted(o, __builtin_amdgcn_exp2f(part_ml[2 * at] - mu), reinterpret_cast<const float4*>(part_o + at * kHd)[lane]);
            }
        }
        const float inv = 1.0f / l;
        *reinterpret_cast<float4*>(out + row * kHd + 4 * lane) = gated(make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv), gate);
    }
}

// One workgroup a CU: up to 256 vector and 216 accumulation registers a lane.
int decode_workgroups(const q35m_ctx* c) { return c->n_cu; }

}  // namespace

size_t paged_decode_work_bytes(const q35m_ctx* c) {
    return (size_t)2 * decode_workgroups(c) * kPagedDecodeHeads * (kHd + 2) * sizeof(float);
}

hipError_t launch_paged_decode(q35m_paged* p, int layer, const PagedBatch& b, const float* q_gate, const float* k,
                               const float* v, float* out) {
    q35m_ctx* c = p->ctx;
    const int per_kv = c->d.nh / c->d.nkv;
    // q heads a workgroup: all of a kv head's up to 16, else 16 or 8 of them.
    const int hg = per_kv <= 16 ? per_kv : per_kv % 16 == 0 ? 16 : 8;
    const int ng = per_kv / hg, nwg = decode_workgroups(c);
    float* part_o = p->work;
    float* part_ml = part_o + (size_t)2 * nwg * kPagedDecodeHeads * kHd;
    const PagedView pv = p->view(layer);
    const AttnLayer& L = c->full[layer];
    // Short sequences that each get a workgroup are not cut, and nothing is to be
    // joined, as the lengths known here say (not so those of a replay): up to 4 units
    // of an fp16 cache (5.7 to 6.5 us against 8 to 10 for 1 to 4 sequences of up to 200
    // rows, 7.6 against 8 at 400), up to 2 of an fp32 one (5.8 against 8.2 at 100 rows;
    // no gain at 200).
    const bool half = p->type == Q35M_KV_F16;
    const int base = half ? kUnitRows<_Float16> : kUnitRows<float>, whole = base * (half ? 4 : 2);
    bool cut = (long)b.n * c->d.nkv * ng > nwg;
    for (int i = 0; i < b.n; ++i) cut |= p->map.length(b.seq[i]) >= whole;
    cut = cut || p->capturing();
    const int unit = cut ? base : whole;
    auto go = [&](auto part, auto merge) {
        {
            ProfScope ps(c, K_PAGED_DECODE);
            hipExtLaunchKernelGGL(part, dim3(nwg), dim3(NT), 0, c->stream, ps.a, ps.b, 0, pv, b, q_gate, k, v, L.q_norm,
                                  L.k_norm, out, part_o, part_ml, hg, ng, unit, c->d.eps);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || !cut) return e;
        ProfScope ps(c, K_PAGED_DECODE_MERGE);
        hipExtLaunchKernelGGL(merge, dim3(c->d.nh, b.n), dim3(MW * kWave), 0, c->stream, ps.a, ps.b, 0, pv, b, part_o,
                              part_ml, q_gate, out, hg, ng, nwg);
        return hipGetLastError();
    };
    if (p->type == Q35M_KV_F16)
        return hg <= 8 ? go(paged_decode<_Float16, true>, paged_decode_merge<_Float16>)
                       : go(paged_decode<_Float16, false>, paged_decode_merge<_Float16>);
    return hg <= 8 ? go(paged_decode<float, true>, paged_decode_merge<float>)
                   : go(paged_decode<float, false>, paged_decode_merge<float>);
}

}  // namespace q35
