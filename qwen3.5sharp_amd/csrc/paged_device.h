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
// token, so the cost is not seen.
__device__ __forceinline__ float4 paged_key_row(float4 x, const double* __restrict__ rope, const float* __restrict__ w,
                                                int lane, double eps) {
    const float4 ww = *reinterpret_cast<const float4*>(w + 4 * lane);
    const int d0 = 4 * (lane & 7);
    double c[4], s[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        c[k] = rope[d0 + k];
        s[k] = rope[kRopeHalf + d0 + k];
    }
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

// Four values rounded to the cache's type, stored as one vector.
__device__ __forceinline__ void store_row4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store_row4(_Float16* p, float4 v) {
    *reinterpret_cast<f16x4*>(p) = f16x4{(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
}

}  // namespace q35
