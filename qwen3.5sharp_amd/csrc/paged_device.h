// Device helpers shared by the paged-cache kernels (gfx950, wave64).
#pragma once

#include <type_traits>

#include "common.h"
#include "paged_cache.h"

namespace q35 {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Page id of entry i of a table row, -1 where it is not mapped.  Ids were
// checked when they were mapped; the bounds here only keep a replayed call,
// whose lengths may have moved past its mapped pages, inside the pool.
__device__ __forceinline__ int page_of(const int* __restrict__ row, int i, int max_pages, int n_pages) {
    const int p = i < max_pages ? row[i] : -1;
    return p < n_pages ? p : -1;
}

// First value of row `r` (position in the sequence) of kv head kvh in page
// `page`; page -1 reads page 0.
template <typename T>
__device__ __forceinline__ size_t row_offset(const PagedView& pv, int page, int kvh, int r) {
    const int in = r & ((1 << pv.page_shift) - 1);
    return ((((size_t)max(page, 0) * pv.nkv + kvh) << pv.page_shift) + in) * kHd;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    return v;
}

// One new K row of a kv head, one wave (lane l: dims 4l .. 4l + 3): the
// rotation and the (1 + w) norm in 64 bits, rounded to fp32.  64 bits because
// an fp16 cache rounds the row a second time: a value whose fp32 arithmetic is
// an ulp off falls on the other side of an fp16 rounding border once in about
// 2^13 values, and such a value is 2^-11 off.  A row is 256 values once per
// token, so the cost is not seen.  c, s: the rotation of dims 4 (lane % 8) ..,
// ww: the norm's weights.
__device__ __forceinline__ float4 paged_key_row(float4 x, const double (&c)[4], const double (&s)[4], float4 ww, int lane,
                                                double eps) {
    const float xs[4] = {x.x, x.y, x.z, x.w};
    const float ws[4] = {ww.x, ww.y, ww.z, ww.w};
    double y[4], ss = 0.0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const double a = xs[k], b = row_xor<8>(xs[k]);
        y[k] = lane < 8 ? a * c[k] - b * s[k] : lane < 16 ? b * s[k] + a * c[k] : a;
        ss += y[k] * y[k];
    }
    const double scale = 1.0 / sqrt(wave_sum(ss) / (double)kHd + eps);
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = y[k] * scale * (1.0 + (double)ws[k]);
    float4 r = make_float4((float)y[0], (float)y[1], (float)y[2], (float)y[3]);
    // The fp32 row as a value of its own: an fp16 cache holds the rounding of
    // what an fp32 cache holds (the compiler would fold the two roundings into
    // one from 64 bits, which differs where the fp32 value is a tie).
    asm volatile("" : "+v"(r.x), "+v"(r.y), "+v"(r.z), "+v"(r.w));
    return r;
}

// With the rotation and the norm weights as they lie in memory.
__device__ __forceinline__ float4 paged_key_row(float4 x, const double* __restrict__ rope, const float* __restrict__ w,
                                                int lane, double eps) {
    const int d0 = 4 * (lane & 7);
    double c[4], s[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        c[k] = rope[d0 + k];
        s[k] = rope[kRopeHalf + d0 + k];
    }
    return paged_key_row(x, c, s, *reinterpret_cast<const float4*>(w + 4 * lane), lane, eps);
}

// Exponent e such that every value of a normed q row, times log2(e) / 16 and
// 2^e, is below 2^15: its fp16 halves are in range whatever the norm weights, and
// hold values from 2^-16 of the bound on to 2^-23 of themselves, smaller ones to 2^-39 of
// it.  |q_d| <= 16 |1 + w_d|.
__device__ __forceinline__ int q_exponent(const float* __restrict__ w, int lane) {
    const float4 a = *reinterpret_cast<const float4*>(w + 4 * lane);
    const float m = fmaxf(fmaxf(fabsf(1.0f + a.x), fabsf(1.0f + a.y)), fmaxf(fabsf(1.0f + a.z), fabsf(1.0f + a.w)));
    const int e = __builtin_amdgcn_frexp_expf(1.4426951f * wave_max(m));
    return 15 - __builtin_amdgcn_readfirstlane(max(min(e, 100), -100));
}

// (a, b) = hi + lo to 2^-23 of each: one conversion of the pair and a fused
// multiply-add for each remainder (a - hi, exact, rounded to fp16).  hi is made a
// value of its own before it is used: where a is a product, the compiler would
// otherwise round it to fp16 in one step for one use and in two for another,
// which differ by an fp16 step now and then.
__device__ __forceinline__ void split16(float a, float b, f16x2& hi, f16x2& lo) {
    uint32_t x = __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b}), y;
    asm("" : "+v"(x));
    asm("v_fma_mixlo_f16 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]\n\t"
        "v_fma_mixhi_f16 %0, %1, -1.0, %3 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
        : "=&v"(y)
        : "v"(x), "v"(a), "v"(b));
    hi = __builtin_bit_cast(f16x2, x);
    lo = __builtin_bit_cast(f16x2, y);
}
// Eight values, as one operand each.
__device__ __forceinline__ void split16(const float* y, f16x8& hi, f16x8& lo) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        f16x2 h, l;
        split16(y[j], y[j + 1], h, l);
        hi[j] = h.x; hi[j + 1] = h.y;
        lo[j] = l.x; lo[j + 1] = l.y;
    }
}

// The output gate's sigmoid, 1 / (1 + e^-g), to fp32 precision: e^-g is 2^t times the
// rounding error of t made good, 1 + d ln 2.  Off by an ulp of the exponential and of
// the reciprocal and by half of one for each of the two sums, 3 ulp in all, whatever g
// is; d is held back for gates so large that t overflows (0 and 1), and NaN stays NaN.
// (e^-g from the rounded product alone is off by |g| 2^-24: 62 half steps at -40.)
// A tile of a prefill takes 64 of them a lane.
__device__ __forceinline__ float gate_sigmoid(float g) {
    const float l2 = 1.44269502e+0f, l2lo = 1.92596303e-8f, ln2 = 0.693147182f;   // log2(e) as a sum, ln 2
    const float t = g * -l2;
    const float d = __builtin_amdgcn_fmed3f(fmaf(g, -l2lo, fmaf(g, -l2, -t)), -1.0f, 1.0f);
    return __builtin_amdgcn_rcpf(fmaf(__builtin_amdgcn_exp2f(t), fmaf(d, ln2, 1.0f), 1.0f));
}
__device__ __forceinline__ float4 gate_sigmoid(float4 g) {
    return make_float4(gate_sigmoid(g.x), gate_sigmoid(g.y), gate_sigmoid(g.z), gate_sigmoid(g.w));
}
// x times it.
__device__ __forceinline__ float4 gated(float4 x, float4 gate) {
    const float4 g = gate_sigmoid(gate);
    return make_float4(x.x * g.x, x.y * g.y, x.z * g.z, x.w * g.w);
}

// Four values rounded to the cache's type, stored as one vector.
__device__ __forceinline__ void store_row4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store_row4(_Float16* p, float4 v) {
    *reinterpret_cast<f16x4*>(p) = f16x4{(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
}

// ---- V values that are not finite -------------------------------------------
//
// The output of a token that sees an infinite V is that infinity, however small the
// weight, and NaN if it sees both or a NaN.  The matrix products cannot say so (0 and
// the low part of a weight times an infinity are NaN, and so are the parts of one), so
// they only have to leave something that is not finite: then, once a segment, the rows
// that its queries see are looked through.  Bits 0 .. 3 of `found`: an infinity or NaN
// in dim 4 lane + bit; bits 4 .. 7: a negative infinity or NaN.
__device__ __forceinline__ bool not_finite(float x) { return !(fabsf(x) < INFINITY); }
__device__ __forceinline__ bool not_finite(_Float16 x) {
    return (__builtin_bit_cast(unsigned short, x) & 0x7c00) == 0x7c00;
}
__device__ __forceinline__ bool not_finite(float4 x) {
    return not_finite(x.x) || not_finite(x.y) || not_finite(x.z) || not_finite(x.w);
}
__device__ __forceinline__ uint32_t infinite(float4 x) {
    auto one = [](float v, int k) { return (v < INFINITY ? 0u : 1u << k) | (v > -INFINITY ? 0u : 16u << k); };
    return one(x.x, 0) | one(x.y, 1) | one(x.z, 2) | one(x.w, 3);
}
__device__ __forceinline__ float4 load_row4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load_row4(const _Float16* p) {
    const f16x4 x = *reinterpret_cast<const f16x4*>(p);
    return make_float4((float)x[0], (float)x[1], (float)x[2], (float)x[3]);
}
// Rows [from, to) of kv head kvh of the sequence whose row of the page table `table` is.
template <typename T>
__device__ __forceinline__ uint32_t infinite_rows(const PagedView& pv, const int* __restrict__ table, int kvh, int from,
                                                  int to, int lane) {
    constexpr int U = 8;       // rows whose loads are in flight together
    uint32_t found = 0;
#pragma nounroll
    for (int r = from; r < to; r += U) {
        float4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int row = min(r + u, to - 1);
            const int page = page_of(table, row >> pv.page_shift, pv.max_pages, pv.n_pages);
            x[u] = load_row4((const T*)pv.v + row_offset<T>(pv, page, kvh, row) + 4 * lane);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) found |= infinite(x[u]);
    }
    return found;
}
__device__ __forceinline__ float4 settled(float4 x, uint32_t found) {
    auto one = [&](float v, int k) {
        const bool up = found >> k & 1, down = found >> k & 16;
        return up ? (!down ? INFINITY : v != v ? v : NAN) : down ? -INFINITY : v;
    };
    return make_float4(one(x.x, 0), one(x.y, 1), one(x.z, 2), one(x.w, 3));
}
// o + f x of a part x of an output, whose infinities stay where f underflows.
__device__ __forceinline__ float4 plus_weighted(float4 o, float f, float4 x) {
    auto one = [&](float a, float v) { return a + (not_finite(v) ? v : f * v); };
    return make_float4(one(o.x, x.x), one(o.y, x.y), one(o.z, x.z), one(o.w, x.w));
}

}  // namespace q35
