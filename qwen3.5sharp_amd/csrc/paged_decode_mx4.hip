// Paged K/V cache in 4 bits: attention of one new token per sequence (paged_decode.hip
// says what is computed and how the rows are dealt out; here as well a unit is 128
// rows, 32 a wave).
//
// S^T = K Q^T takes K as it lies in the cache: the matrix instruction for 4-, 6- and
// 8-bit floats multiplies blocks of 32 values that share a power of two, which is how a
// row is held.  q takes part in the 6-bit type (3 bits of mantissa, up to 7.5): each
// block of 32 dims is cut into six digits of base 16, x = sum d_k 2^{e - 4 k}, |d_k| <= 8, which
// leave 2^-23 of the block's largest value at most, one power of two each.  The digits are columns
// of the operand: 16 of them are four heads by four digits, so a second product brings
// the last two, and the columns of a head are added at the end: a score to fp32 precision
// at two products of 16 x 16 x 128 a head quad, and no K value is converted.
// O^T = V^T P^T takes V as fp16, which holds every value of the cache: a conversion of two
// values an instruction, with the row's power of two in it, and a transposition in
// registers; a block's power of two is per row, along this product's sum, so the
// matrix instruction's own cannot serve here.  P is two fp16 values (hi + lo, to 2^-23 of
// it), which are columns too up to 8 heads.
//
// What bounds it: the cache's bytes and, near to them, the vector work on them.  Calls over caches
// in turn, too many for the last-level cache: 64 sequences of up to 4000 rows are 191 MB, 29 us at the
// 6.5 TB/s that a large read reaches, and take 42 (4.6 TB/s) and the joining 5; 8 of up to 32768 rows, 202
// MB, 39 and 5.  A wave issues vector instructions in 29 % of its cycles, with another one on
// its SIMD, and waits in 30 %.  Two workgroups a CU with a tile ahead each against one with two
// tiles ahead, calls with their rows read back: 51.9 and 48.2 us against 55.9 and 48.1, three short
// sequences 11.6 against 12.2, 32 sequences of up to 6000 rows under 8 heads a kv head (whose loop
// spills 7 registers at two a CU) 39.9 against 37.5; a workgroup's start (lengths, pages, q and the first
// rows, one after the other, 4500 cycles) hides behind the other's rows.  Parts joined by the last
// workgroup to finish instead of by a second launch: 47 us for 43.
#include <algorithm>

#include "paged_decode.h"

namespace q35 {
namespace {

constexpr int NT = 256;
constexpr int kTileRows = 32;                    // of a wave
constexpr int kUnitRows4 = 4 * kTileRows;
constexpr int kDigits = 6;
constexpr int kDigitWords = 50;                  // 48 words of 6-bit codes, and 2 for the banks
// P is 2^{s - m} (s in log2), and m begins kShift4 below the largest score: the output is scaled
// (128 instructions of the tile's 370) only when a score is more than kTop4 above m (the difference is
// compared, as in the fp16 prefill).  Weights are below 2^15.9, in fp16's range, and their low
// halves in steps of 2^-39 of the largest weight or finer, as over an fp16 cache.  Steps of 2^-30
// (kShift4 6) 51.5 us for 64 sequences of up to 4000 rows and 38.8 for 32 of up to 6000 under 16 heads on
// one kv head, 2^-37 (13) 51.7 and 39.4, 2^-39 51.9 and 40.2.
constexpr float kShift4 = 15.0f, kTop4 = 15.9f;

typedef int i32x8 __attribute__((ext_vector_type(8)));

// c += A B for 16 x 16 x 128: A in 4 bits (16 bytes a lane: row l % 16, values 32 (l / 16) ..),
// B in 6 (24 bytes), byte T of the scales.
template <int T>
__device__ __forceinline__ f32x4 scaled_product(u32x4 a, const uint32_t (&b)[6], f32x4 c, uint32_t sa, uint32_t sb) {
    const i32x8 x = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
    const i32x8 y = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], (int)b[4], (int)b[5], 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 2, T, (int)sa, T, (int)sb);
}

// NQ: quads of q heads a workgroup takes, 1, 2 or 4.
template <int NQ>
struct Tile4 {
    static constexpr int kHeads = 4 * NQ;
    uint32_t q[NQ][2][2][6];   // [quad][digits 0 .. 3, 4 ..][t]: head 4 quad + n % 4, digit n / 4 of these, dims 64 g + 32 t ..
    uint32_t qs[NQ][2];        // their scales, byte t
    struct Rows {
        u32x4 kc[2][2];        // row 16 kb + n, dims 64 g + 32 t ..
        uint32_t ks[2];        // its scales of blocks 4 (g / 2) ..
        uint2 vc[8];           // row 16 (j / 4) + 4 g + j % 4, dims 16 n ..
        uint32_t vs[2];        // scales of rows 16 kb + 4 g .., block n / 2
    };
    f32x4 o[16];               // dims 64 g + 16 i + x at [x][i]

    __device__ __forceinline__ void load_q(const uint32_t (*codes)[kDigits][kDigitWords], const uint8_t (*scales)[kDigits][kMxBlocks],
                                           int hg, int lane) {
        const int n = lane & 15, g = lane >> 4;
#pragma unroll
        for (int a = 0; a < NQ; ++a)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int head = min(4 * a + (n & 3), hg - 1), digit = 4 * s + (n >> 2);      // heads from hg on are never read
                const int d = min(digit, kDigits - 1);
                const uint32_t sc = *reinterpret_cast<const uint16_t*>(&scales[head][d][2 * g]);
                qs[a][s] = digit < kDigits ? sc : 0x7f7fu;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int w = 0; w < 6; ++w) q[a][s][t][w] = digit < kDigits ? codes[head][d][12 * g + 6 * t + w] : 0u;
            }
    }
    // (K without the hint that it is read once: an instruction takes half of each line, 48.2 us
    // against 50.4 for 8 sequences of up to 32639 rows.)
    // 16 rows, whose codes begin at `codes` and scales at `scales` (the same for all lanes).
    static __device__ __forceinline__ void load_k(Rows& r, const uint8_t* codes, const uint8_t* scales, int kb, int lane) {
        const int n = lane & 15, g = lane >> 4;
        const uint32_t at = n * kMxCodes + 32 * g, sc = n * kMxBlocks + 4 * (g >> 1);
#pragma unroll
        for (int t = 0; t < 2; ++t) r.kc[kb][t] = *reinterpret_cast<const u32x4*>(codes + at + 16 * t);
        r.ks[kb] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(scales + sc));
    }
    static __device__ __forceinline__ void load_v(Rows& r, const uint8_t* codes, const uint8_t* scales, int kb, int lane) {
        const int n = lane & 15, g = lane >> 4;
        const uint32_t at = 4 * g * kMxCodes + 8 * n, sc = 16 * (n >> 1) + 4 * g;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
            const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(codes + at + i * kMxCodes));
            r.vc[4 * kb + i] = make_uint2(x[0], x[1]);
        }
        r.vs[kb] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(scales + sc));
    }
    // Row `at` of the tile (none if negative) is the new one (its codes and scales at kn, vn);
    // rows from `rows` on are masked: what they hold must not be NaN.
    static __device__ __forceinline__ void fix(Rows& x, const uint8_t* kn, const uint8_t* vn, int at, int rows, int lane) {
        const int n = lane & 15, g = lane >> 4;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            if (16 * kb + n == at) {
#pragma unroll
                for (int t = 0; t < 2; ++t) x.kc[kb][t] = *reinterpret_cast<const u32x4*>(kn + 32 * g + 16 * t);
                x.ks[kb] = *reinterpret_cast<const uint32_t*>(kn + kMxCodes + 4 * (g >> 1));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 16 * kb + 4 * g + i;
                const uint32_t keep = ~(0xffu << 8 * i);
                if (r == at) {
                    x.vc[4 * kb + i] = *reinterpret_cast<const uint2*>(vn + 8 * n);
                    x.vs[kb] = (x.vs[kb] & keep) | (uint32_t)vn[kMxCodes + (n >> 1)] << 8 * i;
                }
                if (r >= rows) x.vs[kb] = (x.vs[kb] & keep) | 127u << 8 * i;
            }
        }
    }
    // Scores of rows row_of(j, g) and the lane's head, n % kHeads.
    __device__ __forceinline__ void scores(const Rows& r, float (&s)[8], int lane) const {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            f32x4 c[NQ];
            const uint32_t ks = r.ks[kb] >> (lane & 16);   // blocks 2 g and 2 g + 1
#pragma unroll
            for (int a = 0; a < NQ; ++a) {
                c[a] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int d = 1; d >= 0; --d) {             // the last digits' products first
                    c[a] = scaled_product<0>(r.kc[kb][0], q[a][d][0], c[a], ks, qs[a][d]);
                    c[a] = scaled_product<1>(r.kc[kb][1], q[a][d][1], c[a], ks, qs[a][d]);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x[NQ];
#pragma unroll
                for (int a = 0; a < NQ; ++a) {             // the digits' columns n, n ^ 4, n ^ 8, n ^ 12
                    x[a] = c[a][i];
                    x[a] += row_xor<8>(x[a]);
                    x[a] += row_ror4(x[a]);
                }
                const bool odd = lane & 4, upper = lane & 8;
                if constexpr (NQ == 1) s[4 * kb + i] = x[0];
                if constexpr (NQ == 2) s[4 * kb + i] = odd ? x[1] : x[0];
                if constexpr (NQ == 4) s[4 * kb + i] = upper ? (odd ? x[3] : x[2]) : (odd ? x[1] : x[0]);
            }
        }
    }
    static __device__ __forceinline__ int row_of(int j, int g) { return 16 * (j >> 2) + 4 * g + (j & 3); }
    __device__ __forceinline__ void pv(const Rows& r, const float (&p)[8], int lane) {
        f16x8 ph, pl;
        split16(p, ph, pl);
        if constexpr (NQ < 4) {                            // columns kHeads .. 2 kHeads - 1 are the low parts
            const u32x4 h = __builtin_bit_cast(u32x4, ph), l = __builtin_bit_cast(u32x4, pl);
            u32x4 b;
#pragma unroll
            for (int w = 0; w < 4; ++w) b[w] = lane & kHeads ? l[w] : h[w];
            ph = __builtin_bit_cast(f16x8, b);
        }
        float unit[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) unit[j] = __uint_as_float((r.vs[j >> 2] >> 8 * (j & 3) & 0xffu) << 23);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            auto byte = [&](auto B) {
                constexpr int b = decltype(B)::value;
                uint32_t x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    x[j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w ? r.vc[j].y : r.vc[j].x, unit[j], b));
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t sel = e ? 0x07060302u : 0x05040100u;
                    const u32x4 a = {__builtin_amdgcn_perm(x[1], x[0], sel), __builtin_amdgcn_perm(x[3], x[2], sel),
                                     __builtin_amdgcn_perm(x[5], x[4], sel), __builtin_amdgcn_perm(x[7], x[6], sel)};
                    const f16x8 av = __builtin_bit_cast(f16x8, a);
                    f32x4& to = o[8 * w + 2 * b + e];
                    if constexpr (NQ == 4) to = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, pl, to, 0, 0, 0);
                    to = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, ph, to, 0, 0, 0);
                }
            };
            byte(std::integral_constant<int, 0>{});
            byte(std::integral_constant<int, 1>{});
            byte(std::integral_constant<int, 2>{});
            byte(std::integral_constant<int, 3>{});
        }
    }
    // The output stays in accumulation registers: without a use there the compiler moves all
    // of it back and forth for the rare scaling.
    __device__ __forceinline__ void pin() {
        asm volatile("" : "+a"(o[0]), "+a"(o[1]), "+a"(o[2]), "+a"(o[3]), "+a"(o[4]), "+a"(o[5]), "+a"(o[6]), "+a"(o[7]));
        asm volatile("" : "+a"(o[8]), "+a"(o[9]), "+a"(o[10]), "+a"(o[11]), "+a"(o[12]), "+a"(o[13]), "+a"(o[14]), "+a"(o[15]));
    }
    __device__ __forceinline__ void scale(float by) {
        pin();
#pragma unroll
        for (int x = 0; x < 16; ++x) o[x] *= by;
        pin();
    }
    // The lane's output values, 4 consecutive dims at a time.
    template <typename F>
    __device__ __forceinline__ void each4(int g, F f) const {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int x = 0; x < 16; x += 4) {
                float y[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    y[k] = o[x + k][i];
                    if constexpr (NQ == 1) y[k] += row_ror4(y[k]);         // (columns n and n + 8 agree)
                    if constexpr (NQ == 2) y[k] += row_xor<8>(y[k]);
                }
                f(64 * g + 16 * i + x, make_float4(y[0], y[1], y[2], y[3]));
            }
    }
};

// Digits of a q row's dims 4 l .., as 6-bit codes (sign, 2 bits of exponent, 3 of mantissa)
// of half a digit, packed along the row, and each block's scales.
__device__ __forceinline__ void put_digits(uint32_t (*codes)[kDigitWords], uint8_t (*scales)[kMxBlocks], float4 x, int lane) {
    auto mag = [](float v) { return __float_as_uint(v) & 0x7fffffffu; };
    uint32_t m = max(max(mag(x.x), mag(x.y)), max(mag(x.z), mag(x.w)));
    m = max(m, row_xor_bits<1>(m));
    m = max(m, row_xor_bits<2>(m));
    m = max(m, row_xor_bits<4>(m));
    const int e = max((int)(m >> 23), 40);                 // every |x| is below 2^{e - 126}
    const float up = __uint_as_float((uint32_t)(256 - e) << 23);
    float t[4] = {x.x * up, x.y * up, x.z * up, x.w * up};
#pragma unroll
    for (int k = 0; k < kDigits; ++k) {
        uint32_t c = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float d = rintf(t[i]);
            t[i] = (t[i] - d) * 16.0f;
            const uint32_t a = (uint32_t)fabsf(d);         // a / 2: codes 4 a up to 2, 8 + 2 a from there to 4
            c |= (min(4 * a, 8 + 2 * a) | (d < 0.0f ? 32u : 0u)) << 6 * i;
        }
        // Four lanes' 24 bits are three words.
        const uint32_t next = row_move<0xF9>(c);           // quad_perm 1 2 3 3
        const int at = lane & 3;
        const uint32_t w = c >> 8 * at | next << (24 - 8 * at);
        if (at < 3) codes[k][3 * (lane >> 2) + at] = w;
        if ((lane & 7) == 0) scales[k][lane >> 3] = m >= 0x7f800000u ? (uint8_t)kMxNan : (uint8_t)(e - 1 - 4 * k);
    }
}

template <int NQ, int N>
__global__ __launch_bounds__(NT, NQ == 4 ? 1 : 2) void paged_decode_mx4(PagedView pv, PagedBatchOf<N> b, const float* __restrict__ q_gate,
                                                          const float* __restrict__ knew, const float* __restrict__ vnew,
                                                          const float* __restrict__ q_norm,
                                                          const float* __restrict__ k_norm, float* __restrict__ out,
                                                          float* __restrict__ part_o, float* __restrict__ part_ml, int hg,
                                                          int ng, int unit, int n_cu, float eps) {
    constexpr int R = kTileRows, H = 4 * NQ, HW = H / 4;   // HW: heads a wave forms and joins
    constexpr int D = NQ == 4 ? 2 : 1;                     // tiles a wave asks for ahead
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int groups = pv.nkv * ng, nh = groups * hg;

    __shared__ __align__(16) float obuf[4][H][kHd];
    __shared__ float ml[4][H][2];
    __shared__ __align__(16) uint8_t newrow[4][2][kMxRow + 8];
    __shared__ __align__(16) uint32_t qcodes[H][kDigits][kDigitWords];
    __shared__ __align__(8) uint8_t qscales[H][kDigits][kMxBlocks];

    __shared__ __align__(16) float norms[2][kHd];          // 1 + q's weights, k's
    norms[0][tid] = 1.0f + q_norm[tid];
    norms[1][tid] = k_norm[tid];
    const Units un = unit ? units_of(pv, b, groups, unit, lane)
                          : units_or_whole(pv, b, groups, unit = kUnitRows4, n_cu, gridDim.x, lane);
    lds_barrier();
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
        const int last16 = pos & ~15, in_page = (1 << pv.page_shift) - 1;

        Tile4<NQ> tl;
#pragma unroll
        for (int x = 0; x < 16; ++x) tl.o[x] = f32x4{0.f, 0.f, 0.f, 0.f};
        // Tiles of the wave: k at first + 4 R k.  All but the last are cached rows alone; the
        // last one may hold the new row, and rows past it.
        const int tiles_mine = first < stop ? (stop - first + 4 * R - 1) / (4 * R) : 0;
        const bool ends = tiles_mine && first + (tiles_mine - 1) * 4 * R + R > pos;
        typename Tile4<NQ>::Rows held[D];                  // tiles whose rows are on their way
        // Rows of tile k (past the wave's last one that again, which costs no traffic: loads that
        // are sometimes left out would all be waited for); their pages are asked for a
        // tile before, by scalar loads, which the vector ones are not waited for with.
        typedef const __attribute__((address_space(4))) int const_int;
        const_int* const ids = (const_int*)(uintptr_t)table;
        int id[2];
        auto group = [&](int k, int kb) { return min(first + 4 * R * min(k, max(tiles_mine, 1) - 1) + 16 * kb, last16); };
        auto ask = [&](int k) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) id[kb] = ids[group(k, kb) >> pv.page_shift];
        };
        size_t at[2];
        int in[2];
        auto place = [&](int k) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                at[kb] = mx_page(pv, id[kb] < pv.n_pages ? id[kb] : -1, kvh);
                in[kb] = group(k, kb) & in_page;
            }
        };
        auto load_k = [&](typename Tile4<NQ>::Rows& r) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const uint8_t* const page = (const uint8_t*)pv.k + at[kb];
                Tile4<NQ>::load_k(r, page + (uint32_t)in[kb] * kMxCodes, page + mx_key_scale(pv, in[kb]), kb, lane);
            }
        };
        auto load_v = [&](typename Tile4<NQ>::Rows& r) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const uint8_t* const page = (const uint8_t*)pv.v + at[kb];
                Tile4<NQ>::load_v(r, page + (uint32_t)in[kb] * kMxCodes, page + mx_value_scale(pv, in[kb], 0), kb, lane);
            }
        };
        // What q's rows and the new row are made of is asked for before K and V, so
        // that they are formed while those are on their way; a wave forms every
        // fourth q row, for all.
        const bool has_new = first <= pos / R * R && pos / R * R < stop && (pos / R * R - first) % (4 * R) == 0;
        // (Asked for by all waves, needed or not: a load that some path leaves out is waited for
        // with those behind it.)
        ask(0);
        float4 xq[HW], xk, xv;
        const float* const q_rows = q_gate + ((size_t)i * nh + y * hg) * 2 * kHd + 4 * lane;
#pragma unroll
        for (int k = 0; k < HW; ++k)
            xq[k] = *reinterpret_cast<const float4*>(q_rows + (size_t)min(wave + 4 * k, hg - 1) * 2 * kHd);
        {
            const size_t from = ((size_t)i * pv.nkv + kvh) * kHd + 4 * lane;
            xk = *reinterpret_cast<const float4*>(knew + from);
            xv = *reinterpret_cast<const float4*>(vnew + from);
        }
        const int id_new = ids[pos >> pv.page_shift], len = ((const_int*)(uintptr_t)pv.lens)[seq];
        double cs[4], sn[4];                     // the rotation of dims 4 (lane % 8) ..
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            cs[k] = pv.rope[(size_t)pos * kRopeDim + 4 * (lane & 7) + k];
            sn[k] = pv.rope[(size_t)pos * kRopeDim + kRopeHalf + 4 * (lane & 7) + k];
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < D; ++k) {
            place(k);
            ask(k + 1);
            load_k(held[k]);
            load_v(held[k]);
        }
        __builtin_amdgcn_sched_barrier(0);

        // q: the rotation, the norm, the scale 1/16 (and log2 e, for exp2).
        const float4 qw = reinterpret_cast<const float4*>(norms[0])[lane];
#pragma unroll
        for (int k = 0; k < HW; ++k) {
            const int r = wave + 4 * k;                    // (rows from hg on: the last one again)
            float x[4] = {xq[k].x, xq[k].y, xq[k].z, xq[k].w}, ss = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float a = x[c], z = row_xor<8>(a), co = (float)cs[c], si = (float)sn[c];
                x[c] = lane < 8 ? a * co - z * si : lane < 16 ? z * si + a * co : a;
                ss += x[c] * x[c];
            }
            const float scale = (kLog2e / 16.0f) / sqrtf(wave_sum(ss) / (float)kHd + eps);
            put_digits(qcodes[r], qscales[r],
                       make_float4(x[0] * (scale * qw.x), x[1] * (scale * qw.y), x[2] * (scale * qw.z), x[3] * (scale * qw.w)),
                       lane);
        }
        // The wave that holds the new row makes it (every head group needs it;
        // one writes it to the page, and none reads it from there).
        if (has_new) {
            const MxLane yk = mx_round(paged_key_row<true>(xk, cs, sn, reinterpret_cast<const float4*>(norms[1])[lane], lane, (double)eps)), yv = mx_round(xv);
            uint8_t* const kn = newrow[wave][0];
            uint8_t* const vn = newrow[wave][1];
            reinterpret_cast<uint16_t*>(kn)[lane] = (uint16_t)yk.codes;
            reinterpret_cast<uint16_t*>(vn)[lane] = (uint16_t)yv.codes;
            if ((lane & 7) == 0) {
                kn[kMxCodes + (lane >> 3)] = (uint8_t)yk.scale;
                vn[kMxCodes + (lane >> 3)] = (uint8_t)yv.scale;
            }
            const int pnew = id_new < pv.n_pages ? id_new : -1;
            if (y % ng == 0 && pnew >= 0 && len < pv.max_rows) {
                mx_put_key((uint8_t*)pv.k + mx_page(pv, pnew, kvh), pv, pos & in_page, yk, lane);
                mx_put_value((uint8_t*)pv.v + mx_page(pv, pnew, kvh), pv, pos & in_page, yv, lane);
            }
        }
        lds_barrier();
        tl.load_q(qcodes, qscales, hg, lane);

        float m_run = -INFINITY, l_run = 0.0f;
        // Tile k, whose rows are r; the ones of tile k + D take their place if `more`.
        auto tile = [&](int k, typename Tile4<NQ>::Rows& r, auto more, int visible) __attribute__((always_inline)) {
            if (decltype(more)::value) {
                place(k + D);
                ask(k + D + 1);
            }
            float s[8];
            tl.scores(r, s, lane);
            if (decltype(more)::value) load_k(r);
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (!decltype(more)::value) s[j] = tl.row_of(j, g) < visible ? s[j] : -INFINITY;
                mx = fmaxf(mx, s[j]);
            }
            mx = xor16_max(xor32_max(mx));
            if (__builtin_expect(__any(mx - m_run > kTop4), 0)) {          // (m_run is -inf at first)
                float m_new = fmaxf(m_run, mx - kShift4);
                if (mx - m_new > kTop4) m_new = mx;        // (mx so large that it is rounded)
                const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.0f : m_new));
                m_run = m_new;
                l_run *= alpha;
                tl.scale(alpha);
            }
            const float sub = m_run == -INFINITY ? 0.0f : -m_run;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                s[j] = __builtin_amdgcn_exp2f(s[j] + sub);
                sum += s[j];
            }
            l_run += sum;
            tl.pv(r, s, lane);
            if (decltype(more)::value) load_v(r);
        };
        const int plain = tiles_mine - (ends ? 1 : 0);
        int k = 0;
#pragma nounroll
        for (; k + D <= plain; k += D) {
#pragma unroll
            for (int d = 0; d < D; ++d) tile(k + d, held[d], std::true_type{}, 0);
        }
        auto last = [&](typename Tile4<NQ>::Rows& r) __attribute__((always_inline)) {
            const int base = first + 4 * R * k;
            Tile4<NQ>::fix(r, newrow[wave][0], newrow[wave][1], pos - base, rows - base, lane);
            tile(k, r, std::false_type{}, rows - base);
        };
        if (D == 2 && k < plain) {
            tile(k, held[0], std::true_type{}, 0);
            ++k;
            if (ends) last(held[D - 1]);
        } else if (ends) {
            last(held[0]);
        }

        // The four waves of the segment join.
        l_run = xor16_sum(xor32_sum(l_run));
        tl.each4(g, [&](int d, float4 x) {
            if (n < hg) *reinterpret_cast<float4*>(&obuf[wave][n][d]) = x;
        });
        if (n < hg && g == 0) {
            ml[wave][n][0] = m_run;
            ml[wave][n][1] = l_run;
        }
        const bool whole = t0 == 0 && t1 == tiles;
        const int slot = 2 * blockIdx.x + (t0 == 0);
        float4 gate[HW];
#pragma unroll
        for (int k = 0; k < HW; ++k)
            if (whole && wave + 4 * k < hg)
                gate[k] = *reinterpret_cast<const float4*>(q_rows + (size_t)(wave + 4 * k) * 2 * kHd + kHd);
        lds_barrier();
        // (A value of the cache that is not finite is NaN, and NaN times any weight is, so
        // nothing is to be settled here.)
#pragma unroll
        for (int k = 0; k < HW; ++k) {
            const int r = wave + 4 * k;
            if (r >= hg) break;
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
            if (whole) {
                const float inv = 1.0f / l;
                *reinterpret_cast<float4*>(out + ((size_t)i * nh + y * hg + r) * kHd + 4 * lane) =
                    gated(make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv), gate[k]);
            } else {
                const size_t at = (size_t)slot * kPagedDecodeHeads + r;
                *reinterpret_cast<float4*>(part_o + at * kHd + 4 * lane) = o;
                if (lane == 0) *reinterpret_cast<float2*>(part_ml + 2 * at) = make_float2(M, l);
            }
        }
        lds_barrier();
    }
}

}  // namespace

hipError_t launch_paged_decode_mx4(q35m_paged* p, int layer, const PagedBatch& b, const float* q_gate, const float* k,
                                   const float* v, float* out) {
    q35m_ctx* c = p->ctx;
    const int per_kv = c->d.nh / c->d.nkv;
    const int hg = per_kv <= 16 ? per_kv : per_kv % 16 == 0 ? 16 : 8;
    // (16 heads take 470 of a lane's 512 registers: one workgroup a CU)
    const int ng = per_kv / hg, nwg = c->n_cu * (hg <= 8 ? 2 : 1);
    float* part_o = p->work;
    float* part_ml = part_o + (size_t)2 * nwg * kPagedDecodeHeads * kHd;
    const PagedView pv = p->view(layer);
    const AttnLayer& L = c->full[layer];
    // (Where the lengths are known here, nothing is launched to join sequences left whole; else the
    // kernels find it: unit 0.)
    int units = 0, longest = 0;
    for (int i = 0; i < b.n; ++i) {
        const int n = p->map.length(b.seq[i]) / kUnitRows4 + 1;
        units += n * c->d.nkv * ng;
        longest = std::max(longest, n);
    }
    const bool known = p->lengths_known(), whole = left_whole(b.n * c->d.nkv * ng, units, longest, c->n_cu, nwg);
    const int unit = !known ? 0 : whole ? kUnitRows4 * longest : kUnitRows4;
    return with_batch(b, [&](const auto& some) {
        constexpr int N = std::decay_t<decltype(some)>::kSeqs;
        {
            ProfScope ps(c, K_PAGED_DECODE);
            auto go = [&](auto kern) {
                hipExtLaunchKernelGGL(kern, dim3(nwg), dim3(NT), 0, c->stream, ps.a, ps.b, 0, pv, some, q_gate, k, v, L.q_norm,
                                      L.k_norm, out, part_o, part_ml, hg, ng, unit, c->n_cu, c->d.eps);
            };
            if (hg <= 4) go(paged_decode_mx4<1, N>);
            else if (hg <= 8) go(paged_decode_mx4<2, N>);
            else go(paged_decode_mx4<4, N>);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || (known && whole)) return e;
        ProfScope ps(c, K_PAGED_DECODE_MERGE);
        hipExtLaunchKernelGGL((paged_decode_merge<kUnitRows4, N>), dim3(c->d.nh, b.n), dim3(MW * kWave), 0, c->stream, ps.a,
                              ps.b, 0, pv, some, part_o, part_ml, q_gate, out, hg, ng, nwg, known ? 0 : c->n_cu);
        return hipGetLastError();
    });
}

}  // namespace q35
