// Products with e4m3 codes under f32 scales: one scale per 128 x 128 block of the weights, one per row and 128 elements
// of the activations. Row quantisation, expert-sorted rows, the products and the weighted combination.
#pragma once
#include <cuda_fp8.h>

#include "cluster.cuh"

namespace oco {

constexpr int kF8MaxExperts = 512, kF8MaxTopK = 16;

// Four f32 values as e4m3 codes in one word (round to nearest even; beyond the range: the largest; NaN stays NaN).
__device__ __forceinline__ uint32_t f8x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

// ---- expert-sorted order of the routes ----------------------------------------------------------------------------
// One cluster of CTAs: each counts the routes of each expert in its share of the ids, all add up the counts of all, then
// every route gets its row. The order inside an expert follows the atomics and may differ from call to call; rows are
// independent and leave through their route, so no result does.
struct F8PlanParams {
    const uint32_t* ids;      // [R]; outside 0 .. E-1: no route of this plan
    uint32_t* offsets;        // [E + 1]
    uint32_t* route_of_row;   // [R]
    uint32_t* row_of_route;   // [R]; 0xffffffff: a route without a row
    uint32_t* tiles;          // pairs (expert, first sorted row), tile_rows rows each
    uint32_t* tile_count;
    int R, E, tile_rows;
};
__global__ void __launch_bounds__(1024) f8_plan_kernel(const F8PlanParams p) {
    pdl_wait();                // the kernel before has completed and its writes are visible
    pdl_launch_dependents();
    __shared__ uint32_t count[kF8MaxExperts], next[kF8MaxExperts], warp_rows[32], warp_tiles[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ctas = (int)cluster_size(), rank = (int)cluster_rank();
    const int per = (p.R + ctas - 1) / ctas, i0 = min(p.R, rank * per), i1 = min(p.R, i0 + per);
    if (tid < kF8MaxExperts) count[tid] = 0;
    __syncthreads();
    for (int i = i0 + tid; i < i1; i += 1024) {
        const uint32_t e = p.ids[i];
        if (e < (uint32_t)p.E) atomicAdd(&count[e], 1u);
    }
    cluster_sync_all();
    // thread e: the routes of expert e, and those in the shares before this one; exclusive scans of rows and tiles
    uint32_t c = 0, before = 0;
    if (tid < p.E)
        for (int q = 0; q < ctas; q++) {
            const uint32_t n = __float_as_uint(peer_f32(smem_u32(&count[tid]), (uint32_t)q));
            if (q < rank) before += n;
            c += n;
        }
    const uint32_t nt = (c + p.tile_rows - 1) / p.tile_rows;
    uint32_t sc = c, st = nt;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, sc, d), b = __shfl_up_sync(0xffffffffu, st, d);
        if (lane >= d) { sc += a; st += b; }
    }
    if (lane == 31) { warp_rows[warp] = sc; warp_tiles[warp] = st; }
    __syncthreads();
    uint32_t r0 = sc - c, t0 = st - nt;
    for (int w = 0; w < min(warp, (kF8MaxExperts + 31) / 32); w++) { r0 += warp_rows[w]; t0 += warp_tiles[w]; }
    if (tid < p.E) {
        next[tid] = r0 + before;
        if (rank == 0) p.offsets[tid] = r0;
        for (uint32_t t = rank; t < nt; t += ctas) { p.tiles[2 * (t0 + t)] = tid; p.tiles[2 * (t0 + t) + 1] = r0 + t * p.tile_rows; }
        if (rank == 0 && tid == p.E - 1) { p.offsets[p.E] = r0 + c; *p.tile_count = t0 + nt; }
    }
    __syncthreads();
    for (int i = i0 + tid; i < i1; i += 1024) {
        const uint32_t e = p.ids[i];
        uint32_t row = 0xffffffffu;
        if (e < (uint32_t)p.E) {
            row = atomicAdd(&next[e], 1u);
            p.route_of_row[row] = (uint32_t)i;
        }
        p.row_of_route[i] = row;
    }
    cluster_sync_all();        // nobody leaves while its counts are read
}

// ---- rows to codes ------------------------------------------------------------------------------------------------
// code = e4m3(x * 448 / largest), the quotient rounded once before e4m3's own rounding, so that an element halfway between
// two codes is decided as such; scale = largest / 448. x * 448 is exact for bf16 x, rounded for activations, which are f32.
// The quotient is the product with the rounded reciprocal, corrected once by its exact residual (Markstein's method: the
// correction of a correctly rounded reciprocal's product rounds correctly while nothing leaves the normal range; a block
// whose largest lies outside 2^-100 .. 2^100 is moved by 2^100 first, which is exact but for elements whose code is 0). One
// path for all: a division for such blocks beside it cost a gated product of few columns a third of its time.
// A block whose largest is NaN or infinite gives NaN codes or a scale that makes its products NaN.
struct F8Divider {
    float top, rcp, lift, back;      // largest * lift, its reciprocal; lift: 1, 2^100 or 2^-100, back: its reciprocal
    __device__ __forceinline__ explicit F8Divider(float largest) {
        constexpr float kUp = 1.2676506e30f, kDown = 7.8886091e-31f;               // 2^100, 2^-100
        lift = largest < kDown ? kUp : largest > kUp ? kDown : 1.0f;
        back = largest < kDown ? kDown : largest > kUp ? kUp : 1.0f;
        top = largest == 0.0f ? 1.0f : largest * lift;
        rcp = __frcp_rn(top);
        if (largest == 0.0f) back = 0.0f;
    }
    // largest / 448, by the same method
    __device__ __forceinline__ float scale() const {
        constexpr float kPart = 1.0f / 448.0f;
        const float q = top * kPart;
        return fmaf(fmaf(-q, 448.0f, top), kPart, q) * back;
    }
    // Two quotients in packed f32 arithmetic.
    __device__ __forceinline__ uint64_t two(uint64_t x) const {
        const float up = 448.0f * lift;
        const uint64_t r2 = f32x2(rcp, rcp), n = mul_f32x2(x, f32x2(up, up)), q = mul_f32x2(n, r2);
        return fma_f32x2(fma_f32x2(q, f32x2(-top, -top), n), r2, q);
    }
    // Four f32 elements -> codes.
    __device__ __forceinline__ uint32_t codes(uint64_t a, uint64_t b) const {
        float v[4];
        f32x2_split(two(a), v[0], v[1]);
        f32x2_split(two(b), v[2], v[3]);
        return f8x4(v[0], v[1], v[2], v[3]);
    }
    // Eight bf16 elements -> codes.
    __device__ __forceinline__ uint2 codes(const uint4& x) const {
        return make_uint2(codes(f32x2_bits(x.x << 16, x.x & 0xffff0000u), f32x2_bits(x.y << 16, x.y & 0xffff0000u)),
                          codes(f32x2_bits(x.z << 16, x.z & 0xffff0000u), f32x2_bits(x.w << 16, x.w & 0xffff0000u)));
    }
};

// N (1 or 2) blocks of 128 bf16 elements of half a warp, eight of each a lane -> codes and scales. All 32 lanes take part.
// The largest magnitude is found on the upper 16 bits of f32 values (for non-negative floats the order of the bits, a NaN
// above everything), two of them in a word: both blocks share the four exchanges.
template <int N>
__device__ __forceinline__ void f8_blocks(const uint4 (&x)[N], uint2 (&codes)[N], float (&scale)[N]) {
    uint32_t m = 0;
#pragma unroll
    for (int b = 0; b < N; b++) {
        constexpr uint32_t kMagnitude = 0x7fff7fffu;
        const uint32_t t = __vmaxu2(__vmaxu2(x[b].x & kMagnitude, x[b].y & kMagnitude), __vmaxu2(x[b].z & kMagnitude, x[b].w & kMagnitude));
        m |= max(t & 0xffffu, t >> 16) << (16 * b);
    }
#pragma unroll
    for (int d = 8; d; d >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, d));
#pragma unroll
    for (int b = 0; b < N; b++) {
        const F8Divider by(__uint_as_float(b ? m & 0xffff0000u : m << 16));
        codes[b] = by.codes(x[b]);
        scale[b] = by.scale();
    }
}

// Rows to codes: half a warp per token and two blocks of 128 elements, eight elements of each a lane (two loads on their
// way). A routed token is read and rounded once and its codes written to the row of each of its routes. Scales lie
// [block][row]. One pass over a grid of all rows: CTAs that loop take 3 us more (8192 rows of 4096: 24 us).
__global__ void __launch_bounds__(256) f8_rows_kernel(const uint16_t* x, const uint32_t* row_of_route, int top_k, int tokens, int K, uint8_t* codes,
                                                      float* scales, int scale_pitch) {
    pdl_wait();                // the kernel before has completed and its writes are visible
    pdl_launch_dependents();   // only now: the next kernel reads weights before it waits for this one
    const int lane = threadIdx.x & 15, npairs = (K + 255) / 256;
    const uint32_t units = (uint32_t)tokens * (uint32_t)npairs, u = blockIdx.x * 16 + (threadIdx.x >> 4);
    const uint32_t token = u / (uint32_t)npairs;
    const int pair = (int)(u - token * (uint32_t)npairs), k = pair * 256 + 8 * lane;
    const uint16_t* src = x + (size_t)token * K + k;
    const bool in[2] = {u < units && k < K, u < units && k + 128 < K};
    uint4 q[2];
#pragma unroll
    for (int b = 0; b < 2; b++) q[b] = in[b] ? *reinterpret_cast<const uint4*>(src + 128 * b) : make_uint4(0, 0, 0, 0);
    uint2 c[2];
    float scale[2];
    const uint32_t mine = row_of_route && u < units && lane < top_k ? row_of_route[(size_t)token * top_k + lane] : token;   // lane r: of route r
    f8_blocks(q, c, scale);
    for (int r = 0; r < top_k; r++) {
        const uint32_t row = __shfl_sync(0xffffffffu, mine, r, 16);
        if (row == 0xffffffffu) continue;
#pragma unroll
        for (int b = 0; b < 2; b++) {
            if (in[b]) *reinterpret_cast<uint2*>(codes + (size_t)row * K + k + 128 * b) = c[b];
            if (lane == 0 && in[b]) scales[(size_t)(2 * pair + b) * scale_pitch + row] = scale[b];
        }
    }
}

// ---- weighted combination --------------------------------------------------------------------------------------------
// out[t] = residual[t] + sum_r prob[t, r] y[t, r], one rounding; routes without an expert of this plan are left out. A
// thread takes eight columns of a row.
__global__ void __launch_bounds__(256) f8_combine_kernel(const float* y, const uint32_t* ids, const float* probs,
                                                         const uint16_t* residual, uint16_t* out, int rows, int top_k, int H, int E) {
    pdl_launch_dependents();   // the next kernel of the step may be set up beside this one
    pdl_wait();                // the kernel before has completed and its writes are visible
    const uint32_t per_row = (uint32_t)H / 8, units = (uint32_t)rows * per_row;
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < units; i += gridDim.x * 256) {
        const uint32_t t = i / per_row, c = (i - t * per_row) * 8;
        const uint4 q = *reinterpret_cast<const uint4*>(residual + (size_t)t * H + c);
        float sum[8] = {};
        for (int r0 = 0; r0 < top_k; r0 += 4) {                        // four routes' rows on their way at a time
            float4 v[4][2];
            float pr[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const bool live = r0 + r < top_k && ids[(size_t)t * top_k + r0 + r] < (uint32_t)E;
                pr[r] = live ? probs[(size_t)t * top_k + r0 + r] : 0.f;
                const float4* from = reinterpret_cast<const float4*>(y + ((size_t)t * top_k + r0 + r) * H + c);
#pragma unroll
                for (int j = 0; j < 2; j++) v[r][j] = live ? from[j] : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    sum[4 * j] = fmaf(pr[r], v[r][j].x, sum[4 * j]);
                    sum[4 * j + 1] = fmaf(pr[r], v[r][j].y, sum[4 * j + 1]);
                    sum[4 * j + 2] = fmaf(pr[r], v[r][j].z, sum[4 * j + 2]);
                    sum[4 * j + 3] = fmaf(pr[r], v[r][j].w, sum[4 * j + 3]);
                }
            }
        }
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(w[j] << 16) + sum[2 * j], __uint_as_float(w[j] & 0xffff0000u) + sum[2 * j + 1]);
            o[j] = *reinterpret_cast<const uint32_t*>(&b);
        }
        *reinterpret_cast<uint4*>(out + (size_t)t * H + c) = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

}  // namespace oco
