// Products with e4m3 codes under f32 scales: one scale per 128 x 128 block of the weights, one per row and 128 elements
// of the activations. Row quantisation, expert-sorted rows, the products and the weighted combination.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace oco {

constexpr int kF8MaxExperts = 512, kF8MaxTopK = 16, kF8Block = 128;

// Four f32 values as e4m3 codes in one word (round to nearest even; beyond the range: the largest; NaN stays NaN).
__device__ __forceinline__ uint32_t f8x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}
__device__ __forceinline__ float f8_value(uint8_t c) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3);
    return __half2float(*reinterpret_cast<const __half*>(&h));
}

// ---- expert-sorted order of the routes ----------------------------------------------------------------------------
// One CTA: counts the routes of each expert, then gives every route its row. The order inside an expert follows the
// atomics and may differ from call to call; rows are independent and leave through their route, so no result does.
struct F8PlanParams {
    const uint32_t* ids;      // [R]; outside 0 .. E-1: no route of this plan
    uint32_t* offsets;        // [E + 1]
    uint32_t* route_of_row;   // [R]
    uint32_t* tiles;          // pairs (expert, first sorted row), tile_rows rows each
    uint32_t* tile_count;
    int R, E, tile_rows;
};
__global__ void __launch_bounds__(1024) f8_plan_kernel(const F8PlanParams p) {
    pdl_launch_dependents();   // the next kernel of the step may be set up beside this one
    pdl_wait();                // the kernel before has completed and its writes are visible
    __shared__ uint32_t count[kF8MaxExperts], next[kF8MaxExperts], warp_rows[32], warp_tiles[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid < kF8MaxExperts) count[tid] = 0;
    __syncthreads();
    for (int i = tid; i < p.R; i += 1024) {
        const uint32_t e = p.ids[i];
        if (e < (uint32_t)p.E) atomicAdd(&count[e], 1u);
    }
    __syncthreads();
    // exclusive scans of rows and tiles over the experts (thread e: expert e)
    const uint32_t c = tid < p.E ? count[tid] : 0u, nt = (c + p.tile_rows - 1) / p.tile_rows;
    uint32_t sc = c, st = nt;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, sc, d), b = __shfl_up_sync(0xffffffffu, st, d);
        if (lane >= d) { sc += a; st += b; }
    }
    if (lane == 31) { warp_rows[warp] = sc; warp_tiles[warp] = st; }
    __syncthreads();
    uint32_t r0 = sc - c, t0 = st - nt;
    for (int w = 0; w < warp; w++) { r0 += warp_rows[w]; t0 += warp_tiles[w]; }
    if (tid < p.E) {
        next[tid] = r0;
        p.offsets[tid] = r0;
        for (uint32_t t = 0; t < nt; t++) { p.tiles[2 * (t0 + t)] = tid; p.tiles[2 * (t0 + t) + 1] = r0 + t * p.tile_rows; }
        if (tid == p.E - 1) { p.offsets[p.E] = r0 + c; *p.tile_count = t0 + nt; }
    }
    __syncthreads();
    for (int i = tid; i < p.R; i += 1024) {
        const uint32_t e = p.ids[i];
        if (e < (uint32_t)p.E) p.route_of_row[atomicAdd(&next[e], 1u)] = (uint32_t)i;
    }
}

// ---- rows to codes ------------------------------------------------------------------------------------------------
// A warp per row and block of 128 elements, four a lane. code = e4m3(x * 448 / largest) with one rounding before e4m3's:
// x * 0.875 is exact for bf16 x, the division rounds correctly and the power of two is exact, so an element halfway
// between two codes is decided as such. Scales lie [block][row].
__global__ void __launch_bounds__(256) f8_rows_kernel(const uint16_t* __restrict__ x, const uint32_t* __restrict__ route_of_row,
                                                      const uint32_t* __restrict__ live_rows, int top_k, int rows, int K,
                                                      uint8_t* __restrict__ codes, float* __restrict__ scales, int scale_pitch) {
    pdl_wait();                // the kernel before has completed and its writes are visible
    pdl_launch_dependents();   // only now: the next kernel reads weights before it waits for this one
    const int lane = threadIdx.x & 31, nkb = (K + 127) / 128;
    const int n = live_rows ? (int)*live_rows : rows;
    for (long long u = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); u < (long long)n * nkb; u += (long long)gridDim.x * 8) {
        const int row = (int)(u / nkb), kb = (int)(u - (long long)row * nkb), k = kb * 128 + 4 * lane;
        const size_t token = route_of_row ? route_of_row[row] / (uint32_t)top_k : (uint32_t)row;
        uint2 q = make_uint2(0, 0);
        if (k < K) q = *reinterpret_cast<const uint2*>(x + token * K + k);
        float v[4] = {__uint_as_float(q.x << 16), __uint_as_float(q.x & 0xffff0000u), __uint_as_float(q.y << 16), __uint_as_float(q.y & 0xffff0000u)};
        // the largest as bits: for non-negative floats the order of the bits, a NaN above everything
        uint32_t m = max(max(__float_as_uint(fabsf(v[0])), __float_as_uint(fabsf(v[1]))), max(__float_as_uint(fabsf(v[2])), __float_as_uint(fabsf(v[3]))));
        m = __reduce_max_sync(0xffffffffu, m);
        const float top = __uint_as_float(m), div = m ? top : 1.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = __fdiv_rn(v[j] * 0.875f, div) * 512.0f;
        if (k < K) *reinterpret_cast<uint32_t*>(codes + (size_t)row * K + k) = f8x4(v[0], v[1], v[2], v[3]);
        if (lane == 0) scales[(size_t)kb * scale_pitch + row] = __fdiv_rn(top, 448.0f);
    }
}

// ---- weighted combination --------------------------------------------------------------------------------------------
// out[t] = residual[t] + sum_r prob[t, r] y[t, r], one rounding; routes without an expert of this plan are left out. A
// thread takes eight columns of a row.
__global__ void __launch_bounds__(256) f8_combine_kernel(const uint16_t* __restrict__ y, const uint32_t* __restrict__ ids, const float* __restrict__ probs,
                                                         const uint16_t* residual, uint16_t* out, int rows, int top_k, int H, int E) {
    pdl_launch_dependents();   // the next kernel of the step may be set up beside this one
    pdl_wait();                // the kernel before has completed and its writes are visible
    const int per_row = H / 8;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)rows * per_row; i += (long long)gridDim.x * 256) {
        const int t = (int)(i / per_row), c = (int)(i - (long long)t * per_row) * 8;
        float acc[8];
        const uint4 q = *reinterpret_cast<const uint4*>(residual + (size_t)t * H + c);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
        float sum[8] = {};
        for (int r = 0; r < top_k; r++) {
            if (ids[(size_t)t * top_k + r] >= (uint32_t)E) continue;
            const float pr = probs[(size_t)t * top_k + r];
            const uint4 v = *reinterpret_cast<const uint4*>(y + ((size_t)t * top_k + r) * H + c);
            const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                sum[2 * j] = fmaf(pr, __uint_as_float(u[j] << 16), sum[2 * j]);
                sum[2 * j + 1] = fmaf(pr, __uint_as_float(u[j] & 0xffff0000u), sum[2 * j + 1]);
            }
        }
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            acc[2 * j] = __uint_as_float(w[j] << 16) + sum[2 * j];
            acc[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u) + sum[2 * j + 1];
            const __nv_bfloat162 b = __floats2bfloat162_rn(acc[2 * j], acc[2 * j + 1]);
            o[j] = *reinterpret_cast<const uint32_t*>(&b);
        }
        *reinterpret_cast<uint4*>(out + (size_t)t * H + c) = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

}  // namespace oco
