// The paged decode kernels' division of work into units of cache rows, and the
// joining of a sequence's parts (paged_decode.hip says how they are dealt out).
#pragma once

#include "paged_device.h"

namespace q35 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// Sums over lanes 0 .. l, by moves within rows of 16 lanes and then of rows' last values.
template <int CTRL, int ROWS>
__device__ __forceinline__ int scan_step(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, true);
}
__device__ __forceinline__ int wave_scan(int v) {
    v = scan_step<0x111, 0xf>(v);          // row_shr 1, 2, 4, 8
    v = scan_step<0x112, 0xf>(v);
    v = scan_step<0x114, 0xf>(v);
    v = scan_step<0x118, 0xf>(v);
    v = scan_step<0x142, 0xa>(v);          // row_bcast 15, to rows 1 and 3
    return scan_step<0x143, 0xc>(v);       // row_bcast 31, to rows 2 and 3
}

// The units of a call's sequences, one sequence a lane: `end` is the number of
// units up to and with the lane's.
struct Units {
    int rows, tiles, end, total;
};
template <int N>
__device__ __forceinline__ Units units_of(const PagedView& pv, const PagedBatchOf<N>& b, int groups, int unit, int lane) {
    Units u;
    // (the row past max_rows of a replayed call that its caller let run over)
    u.rows = lane < b.n ? min(pv.lens[b.seq[lane]] + 1, pv.max_rows) : 0;
    u.tiles = (u.rows + unit - 1) / unit;
    u.end = u.tiles * groups;
    u.end = wave_scan(u.end);
    u.total = __builtin_amdgcn_readlane(u.end, kWave - 1);
    return u;
}

// Whether a 4-bit cache's sequences are left whole, each (sequence, head group) to a
// workgroup, so that nothing is to be joined: where the busiest CU gets up to 3 units
// more than if they are dealt out (a launch against 1.1 us a unit).  450 rows, 4
// units for 1: 10.9 us against 11.1; 16 sequences of 600, 5 for 2: 13.2 against 14.5, of
// 1000, 8 for 2: 16.5 against 15.7; 64 of 3000, as many: 38.9 against 43.7.
__host__ __device__ __forceinline__ bool left_whole(int groups, int units, int longest, int n_cu, int nwg) {
    const int each = (groups <= n_cu ? 1 : 2) * longest;   // (nwg: one or two a CU)
    return groups <= nwg && (each - 4) * n_cu < units;
}
// The units of such a cache, and how many rows one has.
template <int N>
__device__ __forceinline__ Units units_or_whole(const PagedView& pv, const PagedBatchOf<N>& b, int groups, int& unit, int n_cu,
                                                int nwg, int lane) {
    Units u = units_of(pv, b, groups, unit, lane);
    const int longest = __builtin_amdgcn_readfirstlane((int)wave_max((float)u.tiles));
    if (left_whole(b.n * groups, u.total, longest, n_cu, nwg)) {
        unit *= longest;
        u.tiles = lane < b.n;
        u.end = min(lane + 1, b.n) * groups;
        u.total = b.n * groups;
    }
    return u;
}

// The parts of one (sequence, q head), where its units went to several
// workgroups: waves take parts in turn, a lane four dims.  n_cu: 0, or the CUs of a call
// whose sequences may turn out to be whole.
constexpr int MW = 8;      // waves
template <int UNIT, int N = kMaxBatch>
__global__ __launch_bounds__(MW * kWave) void paged_decode_merge(PagedView pv, PagedBatchOf<N> b,
                                                                 const float* __restrict__ part_o,
                                                                 const float* __restrict__ part_ml,
                                                                 const float* __restrict__ q_gate,
                                                                 float* __restrict__ out, int hg, int ng, int nwg, int n_cu) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int groups = pv.nkv * ng, nh = groups * hg;
    const int i = blockIdx.y, head = blockIdx.x, y = head / hg, h = head - y * hg;
    int unit = UNIT;
    const Units un = n_cu ? units_or_whole(pv, b, groups, unit, n_cu, nwg, lane) : units_of(pv, b, groups, UNIT, lane);
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

}  // namespace
}  // namespace q35
