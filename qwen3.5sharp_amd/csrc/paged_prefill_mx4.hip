// Paged K/V cache in 4 bits: attention of chunks of new tokens (paged_prefill.hip says
// what is computed, how the work is divided and how the fp16 kernel, whose shape this
// one has, pipelines its units).
//
// The scores take K as it lies in the cache, from global memory to registers: the
// matrix instruction for 4-, 6- and 8-bit floats, 32 x 32 x 64, multiplies blocks of 32
// values with a power of two each, and runs four times as many products a cycle as the
// fp16 one.  q is cut into kParts parts of the 6-bit type (3 bits of mantissa), each
// the rounding of what the ones before it left, a power of 16 below: five leave 2^-20 of
// the block's largest value at most (2^-22 unless that is within 1 / 32 below a power of two), at
// 5 / 4 of one fp16 product's time where two would be taken.  Five and not six, which would leave
// a sixteenth of that: of the outputs' 6e-7 over normal rows (fp32's sums) q's parts are the less, and
// a unit's products are 52 instead of 56, 240 us against 250 for 512 rows behind 16000, 100.5
// against 103 for 2048 (where q alone decides, small values of a block beside a large one and scores
// of 6, the outputs are off by up to 2.5e-5, six parts' bound being 1.5e-6).
// The output's products are fp16's, with P as hi + lo: a block's power of two is a row's,
// along that product's sum.  V is converted into LDS, once a workgroup, beside products.
//
// What bounds it: the matrix pipe, by the power that it takes, and what one wave a SIMD issues beside
// it.  A unit of 64 x 64 is 52 products a SIMD; on random values in every CU at once the scores'
// take 22.7 ns each, the output's 18.3, and the two in turn 20.9 (14 to 16 on zeros): 1.09 us of the
// 1.48 that it takes.  The pipe is busy 43 % of the cycles, the wave issues vector instructions
// in 34 % and waits in 15 %.  512 rows behind 16000: 226 us, 591 TFLOP/s of the scores and outputs
// in all.  A tile's beginning and end are 33000 cycles, 14 us, one step after the other (a fifth of it
// waits), and a launch's first ones more: 2048 rows, two tiles a workgroup and 33 units, 86 us.
#include <type_traits>

#include "paged_prefill.h"

namespace q35 {
namespace {

constexpr int NT = 256;
constexpr int kParts = 5;

struct Mx4Tile {
    _Float16 v[2][kUnit][kHd];            // (first q's parts, at the end the gates)
    union {
        float4 q[kPagedTileRows * kHd / 4];   // q rows, at the end the output's
        f16x8 p[2][4][4][kWave];          // a wave's weights of two units: operands (hi, lo) of two 16-row steps
    };
    float mx[2][4][32];                   // maxima of two units' halves; at the end sums and maxima
    float w[kHd];                         // 1 + the norm's weights
    uint8_t qscale[2][4][kWave];          // the first part's scales
    int found;                            // values that are not finite
};
static_assert(2 * 4 * kParts * kWave * (sizeof(uint4) + sizeof(uint2)) <= sizeof(Mx4Tile::v), "the parts' room");

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x6 __attribute__((ext_vector_type(6)));
typedef float f32x32 __attribute__((ext_vector_type(32)));

// c += A B for 32 x 32 x 64: A in 4 bits (16 bytes a lane: row l % 32, values 32 (l / 32) ..),
// B in 6 (24 bytes), byte S of A's scales and of B's.
template <int S>
__device__ __forceinline__ f32x16 scaled_product32(u32x4 a, const uint32_t (&b)[6], f32x16 c, uint32_t sa, uint32_t sb) {
    const i32x8 x = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
    const i32x8 y = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], (int)b[4], (int)b[5], 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 4, 2, S, (int)sa, S, (int)sb);
}

// A block of q, dims 2 i and 2 i + 1 in even[i] and odd[i], as parts of 6 bits, 16 and 8
// bytes each at to[16-byte word][lane] and behind; returned is the first part's scale, of
// which a later one's is 4 less than the one's before.  The conversions are written out
// because their results come while they still read: the compiler lets the two share
// registers.
__device__ __forceinline__ uint32_t cut_block(f32x16 even, f32x16 odd, uint4* to, uint2* to2) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kMxBlock / 2; ++i) m = max(m, max(__float_as_uint(even[i]) & 0x7fffffffu, __float_as_uint(odd[i]) & 0x7fffffffu));
    const uint32_t e = max(m >> 23, 40u);                  // every |x| is below 2^{e - 126}, 8 times 2^{e - 129}
#pragma unroll
    for (int k = 0; k < kParts; ++k) {
        const float unit = __uint_as_float((e - 2 - 4 * k) << 23);
        u32x6 part;
        asm("v_cvt_scalef32_2xpk16_fp6_f32 %0, %1, %2, %3" : "=&v"(part) : "v"(even), "v"(odd), "v"(unit));
        to[k * kWave] = make_uint4(part[0], part[1], part[2], part[3]);
        to2[k * kWave] = make_uint2(part[4], part[5]);
        if (k + 1 == kParts) break;
        f32x32 back;
        asm("v_cvt_scalef32_pk32_f32_fp6 %0, %1, %2" : "=&v"(back) : "v"(part), "v"(unit));
#pragma unroll
        for (int i = 0; i < kMxBlock / 2; ++i) {
            even[i] -= back[2 * i];
            odd[i] -= back[2 * i + 1];
        }
    }
    return m >= 0x7f800000u ? kMxNan : e - 2;
}

__global__ __launch_bounds__(NT, 1) void paged_prefill_mx4(PagedView pv, PagedBatch b, const float* __restrict__ q_gate,
                                                           const float* __restrict__ q_norm, float* __restrict__ out,
                                                           float* __restrict__ part_o, float* __restrict__ part_ml,
                                                           int hg_shift, int ng, int more, float eps) {
    // (as in the fp16 kernel)
    constexpr float kShift = 6.0f, kTop = 15.9f;
    __shared__ __align__(16) Mx4Tile st;
    const int tid = threadIdx.x;
    const int tm = kPagedTileRows >> hg_shift;
    const int groups = pv.nkv * ng, nh = groups << hg_shift;
    const int wg = xcd_remap(blockIdx.x, gridDim.x);      // neighbours, which share K and V, on one XCD's L2
    constexpr int kBuf = kUnit * kHd * 2;                 // bytes of a V buffer

    const float w = q_norm[tid];
    const Units un = more < 0 ? units_or_whole(pv, b, groups, hg_shift, gridDim.x, tid & 63)
                              : units_of(pv, b, groups, hg_shift, more, tid & 63);
    st.w[tid] = 1.0f + w;                                 // (read behind the first segment's first barrier)
    Walk wk;
    wk.begin(un, wg, gridDim.x);
    while (wk.next(b, un, groups, hg_shift)) {
        const int start = uniform(wk.start), tokens = uniform(wk.tokens);
        const int seq = b.seq[wk.i], kvh = wk.y / ng;
        const int* table = pv.table + (size_t)seq * pv.max_pages;
        // (the lane's and the wave's own places as values of this segment: addresses made of them
        // would else be kept over all segments, moved out of the registers and back)
        int lane = tid & 63, nn = lane & 31, wave = uniform(tid >> 6);
        asm volatile("" : "+v"(lane), "+v"(nn), "+s"(wave));
        const int h = lane >> 5, rg = wave & 1, half = wave >> 1;
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
        // (Made anew for each use, for the same reason.)
        auto rows_from = [&]() {
            int shift = hg_shift;
            asm volatile("" : "+s"(shift));
            return [=](int r) { return min(r >> shift, left - 1) * nh + (r & ((1 << shift) - 1)); };
        };

        // A wave takes rows 32 half .. of a unit's K and brings rows 16 wave .. of its V,
        // the rg-th 16 of those.  It holds where 64 entries of the page table lie, one a lane,
        // from entry `held` on (one instruction fewer counts here: see above).
        int held = 0;
        uint32_t at_lo = 0, at_hi = 0;                     // of the K page; V's is v_behind further
        const uint64_t v_behind = (uint64_t)pv.v - (uint64_t)pv.k;
        const int in_page = (1 << pv.page_shift) - 1, scales = kMxCodes << pv.page_shift;
        auto hold = [&](int entry) {
            held = entry;
            const uint64_t at = (uint64_t)pv.k + mx_page(pv, page_of(table, entry + lane, pv.max_pages, pv.n_pages), kvh);
            at_lo = (uint32_t)at;
            at_hi = (uint32_t)(at >> 32);
        };
        // First row of the g-th 16 rows of unit t that the wave takes (the last 16, past the end).
        auto group = [&](int t, int g) { return min(t * kUnit + 32 * half + 16 * g, last16); };
        auto hold_unit = [&](int t) {
            if (__builtin_expect(uniform((group(t, 1) >> pv.page_shift) - held) >= kWave, 0)) hold(uniform(group(t, 0) >> pv.page_shift));
        };
        // K: lane (row nn, h) takes blocks 4 h .. of its row; V: 16-byte pieces of two rows,
        // 8 i + lane / 8, block lane % 8.
        u32x4 kc[4], vc[2][2];
        uint32_t ks[2], vs[2][2];                          // (V of two units: they are waited for longest)
        struct Keys {
            const uint8_t *row, *scale;
        };
        auto keys = [&](int t) {
            const int r = min(t * kUnit + 32 * half + (nn & 16), last16), in = r & in_page;
            const int from = 4 * ((r >> pv.page_shift) - held);
            const uint32_t lo = __builtin_amdgcn_ds_bpermute(from, (int)at_lo), hi = __builtin_amdgcn_ds_bpermute(from, (int)at_hi);
            const uint8_t* const at = (const uint8_t*)((uint64_t)hi << 32 | lo);
            return Keys{at + (uint32_t)((in + (nn & 15)) * kMxCodes + 64 * h),
                        at + (uint32_t)(scales + (in + (nn & 15)) * kMxBlocks + 4 * h)};
        };
        auto load_values = [&](int t, u32x4 (&vc)[2], uint32_t (&vs)[2]) {
            const int r = uniform(group(t, rg)), from = uniform((r >> pv.page_shift) - held), in = r & in_page;
            const uint64_t at = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)at_hi, from) << 32 |
                                 (uint32_t)__builtin_amdgcn_readlane((int)at_lo, from)) + v_behind;
            const uint32_t code = (uint32_t)(in * kMxCodes + 16 * lane);
            const uint32_t scale = (uint32_t)(scales + in * kMxBlocks + 16 * (lane & 7) + (lane >> 3));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                vc[i] = from_global<u32x4>((const uint8_t*)at + code + 1024 * i);
                vs[i] = from_global<uint8_t>((const uint8_t*)at + scale + 8 * i);
            }
        };

        // q rows, which have the longest way, 16-byte chunks permuted by row (chunk ^ row % 32).
        const auto q_from = rows_from();
#pragma unroll 4
        for (int r = 16 * wave; r < 16 * wave + 16; ++r)
            dma_nth(0, q_tile, q_from(r) * (2 * kHd * 4) + 16 * (lane ^ (r & 31)), lds_address(&st.q[0]) + r * kHd * 4);
        hold(uniform(group(wk.t0, 0) >> pv.page_shift));
        {
            const Keys k = keys(wk.t0);
#pragma unroll
            for (int s = 0; s < 4; ++s) kc[s] = from_global<u32x4>(k.row + 16 * s);
            ks[0] = from_global<uint32_t>(k.scale);
            load_values(wk.t0, vc[0], vs[0]);
            hold_unit(wk.t0 + 1);
            load_values(wk.t0 + 1, vc[1], vs[1]);
        }
        if (tid == 0) st.found = 0;

        // q: the norm's rows in fp32, then partners cut half of each row's blocks into parts
        // and hand them over: lane (row nn, h) blocks 4 h + s, s = 2 half and 2 half + 1.
        {
            float4* const at = st.q + (32 * rg + nn) * (kHd / 4);
            float x[8][8];
            const float scale = q_row(x, at, pv.rope + (size_t)mine * kRopeDim, st.mx[0], rg, half, lane, eps);
            const float* const w = &st.w[128 * half + 8 * h];
#pragma unroll
            for (int s = 0; s < 8; ++s)
#pragma unroll
                for (int c = 0; c < 8; c += 4) {
                    const float4 v = *reinterpret_cast<const float4*>(&w[16 * s + c]);
                    at[(32 * half + 4 * s + 2 * h + c / 4) ^ nn] = make_float4(x[s][c] * (scale * v.x), x[s][c + 1] * (scale * v.y),
                                                                              x[s][c + 2] * (scale * v.z), x[s][c + 3] * (scale * v.w));
                }
        }
        lds_barrier();
        uint4* const parts = reinterpret_cast<uint4*>(&st.v[0][0][0]) + rg * (4 * kParts * kWave) + lane;
        uint2* const parts2 = reinterpret_cast<uint2*>(reinterpret_cast<uint4*>(&st.v[0][0][0]) + 2 * 4 * kParts * kWave) +
                              rg * (4 * kParts * kWave) + lane;
#pragma nounroll
        for (int s = 2 * half; s < 2 * half + 2; ++s) {
            const float4* const at = st.q + (32 * rg + nn) * (kHd / 4);
            f32x16 even, odd;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const float4 v = at[(8 * (4 * h + s) + c) ^ nn];
                even[2 * c] = v.x; odd[2 * c] = v.y; even[2 * c + 1] = v.z; odd[2 * c + 1] = v.w;
            }
            st.qscale[rg][s][lane] = (uint8_t)cut_block(even, odd, parts + s * (kParts * kWave), parts2 + s * (kParts * kWave));
        }
        lds_barrier();
        uint32_t q[4][kParts][6], qs[kParts];
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int k = 0; k < kParts; ++k) {
                const uint4 x = parts[(s * kParts + k) * kWave];
                const uint2 y = parts2[(s * kParts + k) * kWave];
                q[s][k][0] = x.x; q[s][k][1] = x.y; q[s][k][2] = x.z; q[s][k][3] = x.w;
                q[s][k][4] = y.x; q[s][k][5] = y.y;
            }
        qs[0] = st.qscale[rg][0][lane] | st.qscale[rg][1][lane] << 8 | st.qscale[rg][2][lane] << 16 | (uint32_t)st.qscale[rg][3][lane] << 24;
#pragma unroll
        for (int k = 1; k < kParts; ++k) qs[k] = qs[k - 1] - 0x04040404u;      // (no borrow: a scale is 38 or more)
        lds_barrier();                                     // the parts are read
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
        f32x16 sc[2];                                      // the wave's scores of two units

        // V operands of 16 rows and 32 dims: lane (dim nn, h), rows 4 h + {0..3, 8..11},
        // which the transposing read gathers from lanes of 4 rows x 16 dims.
        uint32_t va[2][4];
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            va[0][d] = lds_address(&st.v[0][32 * half + 4 * h + ((lane >> 2) & 3)][0]) +
                       32 * (8 * half + ((2 * d + ((lane >> 4) & 1)) ^ (2 * ((lane >> 2) & 3)) ^ ((lane >> 2) & 1))) + 8 * ((lane & 3) ^ (2 * half));
            va[1][d] = va[0][d] + (half ? -32 * 512 : 32 * 512);   // the partner's rows
        }
        // Where the lane's converted V goes: row 16 wave + 8 i + lane / 8, chunks 4 (lane % 8) + c
        // of 16 bytes, in place chunk ^ 4 (row % 4) ^ 2 (row % 2) ^ (chunk / 16): the rows that one
        // read touches fall into different banks, and so do the 16 lanes that write together.
        uint32_t vto[4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
            vto[c] = lds_address(&st.v[0][16 * wave + (lane >> 3)][0]) + 64 * ((lane & 7) ^ ((lane >> 3) & 3)) +
                     16 * (c ^ ((lane >> 2) & 1) ^ (2 * ((lane >> 3) & 1)));
        float unit[2];
        // The rows' powers of two; rows that not every query row of the tile sees: see guard_rows
        // (a scale of 0 makes the row's values 0).
        auto units = [&](int t, uint32_t (&vs)[2]) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (__builtin_expect(t * kUnit + kUnit - 1 > first, 0)) {
                    const int r = t * kUnit + 16 * wave + 8 * i + (lane >> 3);
                    if (r >= rows) vs[i] = 0;
                    if (r > first && vs[i] == kMxNan) {
                        vs[i] = 0;
                        st.found = 1;
                    }
                }
                unit[i] = __uint_as_float(vs[i] << 23);
            }
        };
        auto convert = [&](int c, const u32x4 (&vc)[2], int buf) {     // the c-th of eight chunks
            const uint32_t x = vc[c >> 2][c & 3];
            const float u = unit[c >> 2];
            const u32x4 y = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, u, 0)),
                             __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, u, 1)),
                             __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, u, 2)),
                             __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, u, 3))};
            typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
            *(lds_u32x4*)(uintptr_t)(vto[c & 3] + buf * kBuf + (c >> 2) * (8 * kHd * 2)) = y;
        };
        // The products between two barriers, with beside(i) behind the i-th slot of 40: 20 of
        // scores, of which each waits for the one before, and between them, if `left`, the 16 that the unit before has left.  A block's
        // codes are replaced by the next unit's once it is done.
        f16x8 v0[4], v1[4], w0[4], w1[4], h0, l0, h1, l1;
        auto left_over = [&](int i) {
            const f16x8 &a = i < 8 ? v0[i & 3] : v1[i & 3], &b = i < 8 ? (i & 4 ? h0 : l0) : (i & 4 ? h1 : l1);
            o[i & 3] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, o[i & 3], 0, 0, 0);
        };
        auto scores = [&](f32x16& x, uint32_t ks, const uint8_t* next, auto left, auto beside) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < 16; ++k) x[k] = 0.0f;
            auto step = [&](auto S) __attribute__((always_inline)) {
                constexpr int s = decltype(S)::value;
#pragma unroll
                for (int k = kParts - 1; k >= 0; --k) {
                    const int i = kParts * s + kParts - 1 - k;
                    x = scaled_product32<s>(kc[s], q[s][k], x, ks, qs[k]);
                    asm volatile("" : "+a"(x));            // here: left to itself the compiler moves it to its use
                    beside(2 * i);
                    __builtin_amdgcn_sched_barrier(0);
                    if (decltype(left)::value && i < 16) left_over(i);
                    beside(2 * i + 1);
                    __builtin_amdgcn_sched_barrier(0);
                }
                kc[s] = from_global<u32x4>(next + 16 * s);
            };
            step(std::integral_constant<int, 0>{});
            step(std::integral_constant<int, 1>{});
            step(std::integral_constant<int, 2>{});
            step(std::integral_constant<int, 3>{});
        };
        // Whether some row of the tile does not see some row of unit t.
        auto masked = [&](int t) { return t * kUnit + kUnit - 1 > first; };
        auto mask = [&](int t, f32x16& sc) {
            const int lim = mine - (t * kUnit + 32 * half) - 4 * h;
#pragma unroll
            for (int k = 0; k < 16; ++k) sc[k] = 8 * (k >> 2) + (k & 3) <= lim ? sc[k] : -INFINITY;
        };
        // Posts the maximum of the unit's scores.
        auto post = [&](int buf, const f32x16& sc) {
            mx = fmaxf(sc[0], sc[1]);
#pragma unroll
            for (int k = 2; k < 16; ++k) mx = fmaxf(mx, sc[k]);
            mx = xor32_max(mx);
            st.mx[buf][wave][nn] = mx;                      // (both halves the same)
        };
        // The row's maximum over both halves of the unit, which may move the one the
        // weights refer to (known a while before it is done).
        bool moves;
        float sub;                                         // what the weights' exponents have added
        auto meet = [&](float other) {
            mx = fmaxf(mx, other);
            moves = __any(mx - m_run > kTop);              // (m_run is -inf at first)
        };
        float alpha;
        auto move = [&]() {
            alpha = 1.0f;
            if (__builtin_expect_with_probability(moves, 0, 0.99)) {
                float m_new = fmaxf(m_run, mx - kShift);
                if (mx - m_new > kTop) m_new = mx;
                alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.0f : m_new));
                m_run = m_new;
                l_run *= alpha;
            }
            sub = m_run == -INFINITY ? 0.0f : -m_run;
        };
        auto scale = [&]() {                               // (once what refers to the maximum before is added)
            if (__builtin_expect_with_probability(moves, 0, 0.99)) {
                pin();
#pragma unroll
                for (int d = 0; d < 4; ++d) o[d] *= alpha;
                pin();
            }
        };
        f16x8 ph[2], pl[2];
        float p_even = 0.0f, p_sum = 0.0f;                 // (of the unit: one small weight at a time would be lost
                                                           // beside a large sum)
        // The k-th weight is begun, and the one before, whose exponential is there by now, summed
        // and cut; 17 steps are 16 weights.
        float p_next = 0.0f;
        auto weight = [&](int k, const f32x16& sc) {
            const float p = p_next;
            if (k < 16) p_next = __builtin_amdgcn_exp2f(sc[k] + sub);
            if (k == 0) return;
            --k;
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
        auto hand_over = [&](int buf) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                st.p[buf][wave][2 * c][lane] = ph[c];
                st.p[buf][wave][2 * c + 1][lane] = pl[c];
            }
        };
        auto take_over = [&](int buf) {
            h0 = st.p[buf][wave ^ 2][0][lane];
            l0 = st.p[buf][wave ^ 2][1][lane];
            h1 = st.p[buf][wave ^ 2][2][lane];
            l1 = st.p[buf][wave ^ 2][3][lane];
        };
        auto v_read = [&](int buf, int whose, int step, f16x8 (&v)[4]) {
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const uint32_t at = va[whose][d] + buf * kBuf + step * 16 * 512;
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

        {
            // (V's loads before K's, as in the loop: they are waited for in order)
            const Keys next = keys(wk.t0 + 1);
            ks[1] = from_global<uint32_t>(next.scale);
            units(wk.t0, vs[0]);
            scores(sc[0], ks[0], next.row, std::false_type{}, [&](int i) {
                if (i % 2 == 0 && i < 16) convert(i / 2, vc[0], 0);
                if (i == 16) {
                    hold_unit(wk.t0 + 2);
                    load_values(wk.t0 + 2, vc[0], vs[0]);
                }
            });
        }
        if (masked(wk.t0)) mask(wk.t0, sc[0]);
        post(1, sc[0]);
        int t = wk.t0;
        lds_barrier();
        meet(st.mx[1][wave ^ 2][nn]);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            h0[k] = l0[k] = h1[k] = l1[k] = (_Float16)0.0f;
#pragma unroll
            for (int d = 0; d < 4; ++d) v0[d][k] = v1[d][k] = (_Float16)0.0f;
        }
        // Unit t's own rows' products, and all that its partner's need but the weights, which
        // come behind the barrier: those products are left to the next unit, between the
        // scores.  behind() runs among the first products, ahead() with the partner's maxima.
        auto output = [&](int buf, auto behind, auto ahead) __attribute__((always_inline)) {
            hand_over(buf);
            scale();
            __builtin_amdgcn_sched_barrier(0);
            behind();
            __builtin_amdgcn_sched_barrier(0);
            lds_barrier();                                 // the partner's weights and maxima
            const float other = st.mx[buf][wave ^ 2][nn];
            take_over(buf);
            __builtin_amdgcn_sched_barrier(0);
            add(w1, ph[1], pl[1]);
            ahead(other);
            __builtin_amdgcn_sched_barrier(0);
        };
        // One barrier a unit: behind it a unit's V, weights and maxima are there, and every wave
        // has read the V before, whose buffer the next one's goes to.  (B: the unit's V buffer and
        // place among the scores; units in pairs, so that what one leaves to the next stays
        // where it is.)
        auto go_on = [&](auto B) __attribute__((always_inline)) {
            constexpr int b = decltype(B)::value;
            const Keys next = keys(t + 2);
            ks[b] = from_global<uint32_t>(next.scale);
            units(t + 1, vs[b ^ 1]);
            move();
            scores(sc[b ^ 1], ks[b ^ 1], next.row, std::true_type{}, [&](int i) {
                if (i % 2 == 0 && i < 34) weight(i / 2, sc[b]);
                if (i % 4 == 1 && i < 32) convert(i / 4, vc[b ^ 1], b ^ 1);
                if (i == 17) v_read(b, 1, 0, v0);
                if (i == 21) v_read(b, 0, 0, w0);
                if (i == 25) v_read(b, 0, 1, w1);
                if (i == 33) v_read(b, 1, 1, v1);
                if (i == 34) {
                    hold_unit(t + 3);
                    load_values(t + 3, vc[b ^ 1], vs[b ^ 1]);
                }
            });
            output(
                b,
                [&]() {
#pragma unroll
                    for (int d = 0; d < 4; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(w0[d], pl[0], o[d], 0, 0, 0);
                    asm volatile("" : "+v"(sc[b ^ 1]));    // in vector registers, where the weights want them
                    if (masked(t + 1)) {
                        asm volatile("");                  // a branch, not selects
                        mask(t + 1, sc[b ^ 1]);
                    }
#pragma unroll
                    for (int d = 0; d < 4; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(w0[d], ph[0], o[d], 0, 0, 0);
                    post(b, sc[b ^ 1]);
                },
                meet);
        };
        const bool whole = wk.t0 == 0 && wk.t1 == wk.tiles;
        auto finish = [&](auto B) __attribute__((always_inline)) {
            constexpr int b = decltype(B)::value;
            move();
            v_read(b, 0, 0, w0);
            v_read(b, 0, 1, w1);
#pragma unroll
            for (int i = 0; i < 17; ++i) {
                if (i < 16) left_over(i);
                weight(i, sc[b]);
                __builtin_amdgcn_sched_barrier(0);
            }
            v_read(b, 1, 0, v0);
            v_read(b, 1, 1, v1);
            output(b, [&]() { add(w0, ph[0], pl[0]); }, [](float) {});
            if (whole) {                                   // the gates of the wave's rows 16 wave .. take V's place
                const auto gate_from = rows_from();
#pragma unroll 4
                for (int r = 16 * wave; r < 16 * wave + 16; ++r)
                    dma_nth(0, q_tile, gate_from(r) * (2 * kHd * 4) + 4 * kHd + 16 * lane, lds_address(&st.v[0][0][0]) + r * kHd * 4);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) left_over(i);
        };
#pragma nounroll
        for (; t + 2 < wk.t1; ++t) {
            go_on(std::integral_constant<int, 0>{});
            ++t;
            go_on(std::integral_constant<int, 1>{});
        }
        if (t + 1 < wk.t1) {
            go_on(std::integral_constant<int, 0>{});
            finish(std::integral_constant<int, 1>{});
        } else {
            finish(std::integral_constant<int, 0>{});
        }
        pin();

        // The tile's rows to LDS, then a row a wave at a time: finished, or as a part
        // to the workspace.  (Places again as values of this part: kept from the
        // segment's beginning they would be in registers all the while.)
        asm volatile("" : "+v"(lane), "+v"(nn), "+s"(wave));
        const int slot = 2 * wg + (wk.t0 == 0);
        l_run = xor32_sum(l_run);
        if (lane < 32) st.mx[1][wave][nn] = l_run;
        if (half == 0 && lane < 32) st.mx[0][rg][nn] = m_run;
        lds_barrier();                                     // the weights are read
        float4* const os = st.q;
        put_rows(os, o, rg, half, lane);
        lds_barrier();
        const int row = 16 * wave + (lane & 15);           // a row's sum and maximum in lane row % 16
        const float l = st.mx[1][row >> 5][row & 31] + st.mx[1][2 + (row >> 5)][row & 31];
        float* const to_part = part_o + (size_t)slot * kPagedTileRows * kHd;
        const auto from_row0 = rows_from();
        auto gate_row = [&](int r) { return q_tile + (uint32_t)(from_row0(r) * (2 * kHd * 4) + 4 * kHd + 16 * lane); };
        auto out_row = [&](int r) { return r >> hg_shift < left ? out_tile + (uint32_t)(from_row0(r) * (kHd * 4) + 16 * lane) : nullptr; };
        dma_wait();                                        // (the gates, which the wave itself has brought)
        auto gate_of = [&](int k) { return reinterpret_cast<const float4*>(&st.v[0][0][0])[(16 * wave + k) * (kHd / 4) + lane]; };
        const bool look = leave_rows(os, l, st.mx[0][row >> 5][row & 31], whole, gate_of, to_part,
                                     part_ml + (size_t)2 * slot * kPagedTileRows, wave, lane, out_row);
        if (__builtin_expect(look || uniform(st.found), 0))
            settle_rows<Mx4>(os, pv, table, kvh, wk.t0 * kUnit, min(rows, wk.t1 * kUnit), first, left, hg_shift, l, whole,
                            to_part, wave, lane, gate_row, out_row);
        lds_barrier();                                     // (the stores need no wait)
    }
}

}  // namespace

PagedPrefillKernel paged_prefill_mx4_kernel() { return paged_prefill_mx4; }

}  // namespace q35
