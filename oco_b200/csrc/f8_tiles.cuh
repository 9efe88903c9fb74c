// Products of e4m3 codes on the tensor cores (tcgen05.mma.kind::f8f6f4), with one f32 scale per row and 128 elements of
// the activations and one per 128 x 128 block of the weights:
//
//     y[row][f] = sum over blocks kb of (xs[kb][row] * ws[f / 128][kb]) * (sum of 128 products of codes)
//
// The inner sums run in tensor memory; after every block of 128 the accumulator is read out, scaled and added to f32
// sums in registers, while the MMAs of the next block fill the other half of tensor memory. Both operands travel by TMA
// (128-byte rows, 128-byte swizzle): no thread touches a code.
//
// f8_wide_kernel: many rows. Rows are the M side (a thread of the epilogue owns one row: its scale is one number, and a
// row's 128 activations lie in two threads), 256 features the N side.
// f8_thin_kernel: few rows. Weights are the M side (128 features), up to 64 rows the N side, so that the weights, which
// are all that has to be read, stream past a narrow tile; a contraction is split over the CTAs of a cluster and joined
// through distributed shared memory, in a fixed order.
//
// Every wait is bounded (mbar_wait); one that gives up sets the status word and the kernel runs on to its end.
#pragma once
#include "f8.cuh"
#include "gemm.cuh"

namespace oco {

struct F8TileParams {
    const float* row_scales;        // [K blocks][pitch]
    const float* s0;                // [experts][ceil(n / 128)][K blocks]: gate (gated) or the one matrix
    const float* s1;                // up (gated)
    const uint32_t* tiles;          // (expert, first sorted row) pairs; null: dense
    const uint32_t* tile_count;
    const uint32_t* offsets;
    const uint32_t* route_of_row;   // result rows (not gated); null: in place
    uint16_t* out;                  // bf16 [..][n]
    uint8_t* codes;                 // gated: codes of the activations [row][n]
    float* code_scales;             // and their scales [ceil(n / 128)][pitch]
    uint32_t* status;
    int n, K, rows, pitch;
};

__device__ __forceinline__ float silu_times(float g, float u) { return sigmoid_times(g, 1.0f) * g * u; }
// Scale and factor of a block of activations whose largest magnitude is `top`: code = e4m3(a * lift * factor). `lift`
// keeps 448 / top finite where top is tiny.
__device__ __forceinline__ void f8_act_scale(float top, float& scale, float& lift, float& factor) {
    lift = top < 1e-30f ? 1.2676506e30f : 1.0f;
    factor = top == 0.0f ? 1.0f : __fdividef(448.0f, top * lift);
    scale = top * (1.0f / 448.0f);
}

// ---- many rows --------------------------------------------------------------------------------------------------------
struct F8Wide {
    static constexpr int kStages = 4, kA = 128 * 128, kB = 256 * 128, kStage = kA + kB;
    static constexpr int kTmaWarp = 8, kMmaWarp = 9, kThreads = 320;
    static constexpr int kCtrl = 256 + 2 * 128 * 4;
    static constexpr int kSmem = kStages * kStage + kCtrl + 1024;
};
// GATED: the 256 columns of a tile are 128 gate and the same 128 up features, the result is silu(gate) * up as codes.
template <bool GATED>
__global__ void __launch_bounds__(F8Wide::kThreads, 1) f8_wide_kernel(const F8TileParams p, const __grid_constant__ CUtensorMap rows_map,
                                                                     const __grid_constant__ CUtensorMap w0_map, const __grid_constant__ CUtensorMap w1_map) {
    using S = F8Wide;
    extern __shared__ unsigned char smem_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t ctrl = base + S::kStages * S::kStage;
    auto full = [&](int s) { return ctrl + 8u * s; };
    auto empty = [&](int s) { return ctrl + 8u * (S::kStages + s); };
    auto tfull = [&](int b) { return ctrl + 8u * (2 * S::kStages + b); };
    auto tempty = [&](int b) { return ctrl + 8u * (2 * S::kStages + 2 + b); };
    uint32_t* slot = reinterpret_cast<uint32_t*>(gen + S::kStages * S::kStage + 8 * (2 * S::kStages + 4));
    volatile uint32_t* abort_flag = slot + 1;
    uint32_t* tops = reinterpret_cast<uint32_t*>(gen + S::kStages * S::kStage + 256);   // [2][128]
    if (tid == 0) {
        for (int s = 0; s < S::kStages; s++) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        for (int b = 0; b < 2; b++) { mbar_init(tfull(b), 1); mbar_init(tempty(b), 8); }
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == S::kMmaWarp) { tmem_alloc(smem_u32(slot), 512); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    pdl_wait();                // the kernel before has completed and its writes are visible
    pdl_launch_dependents();

    constexpr int kFeat = GATED ? 128 : 256;
    const int nfeat = (p.n + kFeat - 1) / kFeat, nkb = (p.K + 127) / 128, nfb = (p.n + 127) / 128;
    const int ntiles = p.tiles ? (int)*p.tile_count : (p.rows + 127) / 128;
    const int total = ntiles * nfeat;
    struct Item { int expert, row0, nv, f0; };
    auto item_of = [&](int i) {
        Item r;
        const int t = i / nfeat;
        r.f0 = (i - t * nfeat) * kFeat;
        if (p.tiles) {
            r.expert = (int)p.tiles[2 * t];
            r.row0 = (int)p.tiles[2 * t + 1];
            r.nv = min(128, (int)p.offsets[r.expert + 1] - r.row0);
        } else {
            r.expert = 0; r.row0 = t * 128; r.nv = min(128, p.rows - r.row0);
        }
        return r;
    };

    if (warp < 8) {
        // ===== epilogue: thread = row (32 * (warp & 3) + lane), half of the columns (warp >> 2) ====================
        const int erow = (warp & 3) * 32 + lane, half = warp >> 2;
        const uint32_t taddr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t col0 = GATED ? 64u * half : 128u * half, col1 = GATED ? 128u + 64u * half : 128u * half + 64u;
        int g = 0;
        for (int i = blockIdx.x; i < total; i += gridDim.x) {
            const Item it = item_of(i);
            const float* xs = p.row_scales + min(it.row0 + erow, p.pitch - 1);
            const int fb = it.f0 / 128 + (GATED ? 0 : min(half, nfb - 1 - it.f0 / 128));
            const float* ws0 = p.s0 + ((size_t)it.expert * nfb + fb) * nkb;
            const float* ws1 = GATED ? p.s1 + ((size_t)it.expert * nfb + fb) * nkb : ws0;
            uint64_t acc[64];
#pragma unroll
            for (int j = 0; j < 64; j++) acc[j] = 0;
            float x1 = xs[0], x2 = nkb > 1 ? xs[p.pitch] : 0.f, a1 = ws0[0], a2 = nkb > 1 ? ws0[1] : 0.f;
            float b1 = GATED ? ws1[0] : 0.f, b2 = GATED && nkb > 1 ? ws1[1] : 0.f;
            for (int kb = 0; kb < nkb; kb++, g++) {
                const float s0 = x1 * a1, s1 = GATED ? x1 * b1 : s0;
                x1 = x2; a1 = a2; b1 = b2;
                if (kb + 2 < nkb) {
                    x2 = xs[(size_t)(kb + 2) * p.pitch];
                    a2 = ws0[kb + 2];
                    if (GATED) b2 = ws1[kb + 2];
                }
                const int b = g & 1;
                if (lane == 0) mbar_wait(tfull(b), (uint32_t)(g >> 1) & 1u, abort_flag, p.status);
                __syncwarp();
                tc_fence_after();
                const uint64_t t0 = f32x2(s0, s0), t1 = f32x2(s1, s1);
#pragma unroll
                for (int h = 0; h < 4; h++) {                         // 32 columns in registers at a time, beside 128 sums
                    uint32_t r[32];
                    tmem_ld32(taddr + 256u * b + (h < 2 ? col0 : col1) + 32u * (h & 1), r);
                    tmem_ld_wait();
                    if (h == 3) {                                     // all of it is in registers: the buffer is free
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(tempty(b));
                    }
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        acc[16 * h + j] = fma_f32x2(f32x2_bits(r[2 * j], r[2 * j + 1]), h < 2 ? t0 : t1, acc[16 * h + j]);
                }
            }
            const bool live = erow < it.nv;
            if (GATED) {
                const int f = it.f0 + 64 * half;                      // this thread's 64 features
                uint32_t top = 0;
#pragma unroll
                for (int j = 0; j < 32; j++) {
                    float g0, g1, u0, u1;
                    f32x2_split(acc[j], g0, g1);
                    f32x2_split(acc[32 + j], u0, u1);
                    const bool in = f + 2 * j < p.n;
                    const float v0 = in ? silu_times(g0, u0) : 0.f, v1 = in ? silu_times(g1, u1) : 0.f;
                    top = max(top, max(__float_as_uint(fabsf(v0)), __float_as_uint(fabsf(v1))));
                    acc[j] = f32x2(v0, v1);
                }
                tops[half * 128 + erow] = top;
                asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");       // the two warps that share the rows
                top = max(top, tops[(half ^ 1) * 128 + erow]);
                asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
                float scale, lift, factor;
                f8_act_scale(__uint_as_float(top), scale, lift, factor);
                if (live) {
                    const size_t row = (size_t)it.row0 + erow;
                    if (half == 0) p.code_scales[(size_t)(it.f0 / 128) * p.pitch + row] = scale;
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        uint32_t w[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            float v[4];
                            f32x2_split(acc[8 * c + 2 * k], v[0], v[1]);
                            f32x2_split(acc[8 * c + 2 * k + 1], v[2], v[3]);
#pragma unroll
                            for (int e = 0; e < 4; e++) v[e] = v[e] * lift * factor;
                            w[k] = f8x4(v[0], v[1], v[2], v[3]);
                        }
                        if (f + 16 * c < p.n) *reinterpret_cast<uint4*>(p.codes + row * p.n + f + 16 * c) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            } else if (live) {
                const int f = it.f0 + 128 * half;
                const size_t row = p.route_of_row ? p.route_of_row[it.row0 + erow] : (uint32_t)(it.row0 + erow);
#pragma unroll
                for (int c = 0; c < 16; c++) {
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        float v0, v1;
                        f32x2_split(acc[4 * c + k], v0, v1);
                        const __nv_bfloat162 o = __floats2bfloat162_rn(v0, v1);
                        w[k] = *reinterpret_cast<const uint32_t*>(&o);
                    }
                    if (f + 8 * c < p.n) *reinterpret_cast<uint4*>(p.out + row * p.n + f + 8 * c) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
    } else if (warp == S::kTmaWarp) {
        if (lane == 0) {
            int g = 0;
            for (int i = blockIdx.x; i < total; i += gridDim.x) {
                const Item it = item_of(i);
                const int wrow = it.expert * p.n + it.f0;
                for (int kb = 0; kb < nkb; kb++, g++) {
                    const int s = g % S::kStages;
                    mbar_wait(empty(s), ((uint32_t)(g / S::kStages) & 1u) ^ 1u, abort_flag, p.status);
                    if (*abort_flag) break;
                    const uint32_t at = base + (uint32_t)s * S::kStage;
                    mbar_arrive_expect_tx(full(s), S::kStage);
                    tma_load_2d(at, &rows_map, kb * 128, it.row0, full(s));
                    tma_load_2d(at + S::kA, &w0_map, kb * 128, wrow, full(s));
                    tma_load_2d(at + S::kA + S::kB / 2, GATED ? &w1_map : &w0_map, kb * 128, GATED ? wrow : wrow + 128, full(s));
                }
                if (*abort_flag) break;
            }
            if (*abort_flag)
                for (int k = max(0, g - S::kStages); k < g; k++) mbar_drain(full(k % S::kStages), (uint32_t)(k / S::kStages) & 1u);
        }
    } else if (lane == 0) {
        const uint32_t idesc = umma_idesc_f16(256);                  // e4m3 x e4m3, f32, M = 128, N = 256
        int g = 0;
        for (int i = blockIdx.x; i < total; i += gridDim.x) {
            for (int kb = 0; kb < nkb; kb++, g++) {
                const int s = g % S::kStages, b = g & 1;
                mbar_wait(tempty(b), ((uint32_t)(g >> 1) & 1u) ^ 1u, abort_flag, p.status);
                mbar_wait(full(s), (uint32_t)(g / S::kStages) & 1u, abort_flag, p.status);
                if (*abort_flag) break;
                tc_fence_after();
                const uint64_t a = umma_desc(base + (uint32_t)s * S::kStage), w = umma_desc(base + (uint32_t)s * S::kStage + S::kA);
#pragma unroll
                for (int k = 0; k < 4; k++) umma_f8f6f4(tmem + 256u * b, a + 2u * k, w + 2u * k, idesc, k ? 1u : 0u);
                umma_commit(empty(s));
                umma_commit(tfull(b));
            }
            if (*abort_flag) break;
        }
        if (*abort_flag && g > 0) mbar_drain(tfull((g - 1) & 1), (uint32_t)((g - 1) >> 1) & 1u);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == S::kMmaWarp) tmem_dealloc(tmem, 512);
}

// ---- few rows ---------------------------------------------------------------------------------------------------------
template <int NT, bool GATED>
struct F8Thin {
    static constexpr int kA = 128 * 128, kMats = GATED ? 2 : 1, kB = NT * 128, kStage = kMats * kA + kB;
    static constexpr int kRoom = 108 * 1024;                            // two CTAs on an SM
    static constexpr int kStages = kRoom / kStage;
    static constexpr int kBufs = 2, kTmemUsed = kBufs * kMats * NT;
    static constexpr int kTmem = kTmemUsed <= 32 ? 32 : kTmemUsed <= 64 ? 64 : kTmemUsed <= 128 ? 128 : 256;
    static constexpr int kTmaWarp = 4, kMmaWarp = 5, kThreads = 192;
    static constexpr int kCtrl = 512;
    static constexpr int kSmem = kStages * kStage + kCtrl + 1024;
    static_assert(kMats * NT * 128 * 4 <= kStages * kStage, "the parts of a split contraction lie where the stages were");
    static_assert(8 * (2 * kStages + 2 * kBufs) + 8 <= 256, "barriers");
};
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float peer_f32(uint32_t local, uint32_t rank) {      // this CTA's shared address `local`, in CTA `rank`
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(local), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

// One item (a tile of up to NT rows of one expert, 128 features) per cluster; CTA r of its S takes the blocks
// [r * per, ..) of the contraction. x = S * (item), items: feature tile fastest.
template <int NT, bool GATED>
__global__ void __launch_bounds__(F8Thin<NT, GATED>::kThreads) f8_thin_kernel(const F8TileParams p, const __grid_constant__ CUtensorMap rows_map,
                                                                             const __grid_constant__ CUtensorMap w0_map,
                                                                             const __grid_constant__ CUtensorMap w1_map) {
    using S = F8Thin<NT, GATED>;
    constexpr int MATS = S::kMats;
    extern __shared__ unsigned char smem_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t ctrl = base + S::kStages * S::kStage;
    auto full = [&](int s) { return ctrl + 8u * s; };
    auto empty = [&](int s) { return ctrl + 8u * (S::kStages + s); };
    auto tfull = [&](int b) { return ctrl + 8u * (2 * S::kStages + b); };
    auto tempty = [&](int b) { return ctrl + 8u * (2 * S::kStages + S::kBufs + b); };
    uint32_t* slot = reinterpret_cast<uint32_t*>(gen + S::kStages * S::kStage + 8 * (2 * S::kStages + 2 * S::kBufs));
    volatile uint32_t* abort_flag = slot + 1;
    uint32_t* tops = reinterpret_cast<uint32_t*>(gen + S::kStages * S::kStage + 256);   // [2][4]
    const int split = (int)cluster_size(), rank = (int)cluster_rank();
    const int nfeat = (p.n + 127) / 128, nkb = (p.K + 127) / 128, per = (nkb + split - 1) / split;
    const int kb0 = min(nkb, rank * per), kb1 = min(nkb, kb0 + per);
    const int item = (int)blockIdx.x / split, tile = item / nfeat, f0 = (item - tile * nfeat) * 128;
    if (tid == 0) {
        for (int s = 0; s < S::kStages; s++) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        for (int b = 0; b < S::kBufs; b++) { mbar_init(tfull(b), 1); mbar_init(tempty(b), 4); }
        *abort_flag = 0;
        fence_barrier_init();
    }
    // a dense product's weights are known already: their first tiles travel while the kernel before still runs
    const bool early = p.tiles == nullptr;
    if (warp == S::kMmaWarp) { tmem_alloc(smem_u32(slot), S::kTmem); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    auto load_weights = [&](int kb, int s, int expert) {
        const uint32_t at = base + (uint32_t)s * S::kStage;
        mbar_arrive_expect_tx(full(s), S::kStage);
        tma_load_2d(at, &w0_map, kb * 128, expert * p.n + f0, full(s));
        if (GATED) tma_load_2d(at + S::kA, &w1_map, kb * 128, expert * p.n + f0, full(s));
    };
    const int first = min(S::kStages, kb1 - kb0);                       // stages filled before anything is waited for
    if (early && warp == S::kTmaWarp && lane == 0)
        for (int k = 0; k < first; k++) load_weights(kb0 + k, k, 0);
    pdl_wait();                // the kernel before has completed and its writes are visible
    pdl_launch_dependents();
    int expert = 0, row0 = tile * NT, nv = min(NT, p.rows - row0);
    if (p.tiles) {
        if (tile >= (int)*p.tile_count) nv = 0;                         // the whole cluster
        else {
            expert = (int)p.tiles[2 * tile];
            row0 = (int)p.tiles[2 * tile + 1];
            nv = min(NT, (int)p.offsets[expert + 1] - row0);
        }
    }
    if (nv > 0) {
        if (warp < 4) {
            // ===== thread = feature, columns = rows ===============================================================
            const uint32_t taddr = tmem + ((uint32_t)(warp * 32) << 16);
            const float* ws0 = p.s0 + ((size_t)expert * nfeat + f0 / 128) * nkb;
            const float* ws1 = GATED ? p.s1 + ((size_t)expert * nfeat + f0 / 128) * nkb : ws0;
            constexpr int L = (NT + 31) / 32;                           // row scales a lane holds
            float acc[MATS][NT], x1[L], x2[L], a1 = 0.f, a2 = 0.f, b1 = 0.f, b2 = 0.f;
#pragma unroll
            for (int m = 0; m < MATS; m++)
#pragma unroll
                for (int c = 0; c < NT; c++) acc[m][c] = 0.f;
            auto fetch = [&](int kb, float (&x)[L], float& a, float& b) {
                if (kb >= kb1) return;
#pragma unroll
                for (int l = 0; l < L; l++) x[l] = p.row_scales[(size_t)kb * p.pitch + min(row0 + 32 * l + (NT < 32 ? lane % NT : lane), p.pitch - 1)];
                a = ws0[kb];
                if (GATED) b = ws1[kb];
            };
            fetch(kb0, x1, a1, b1);
            fetch(kb0 + 1, x2, a2, b2);
            for (int kb = kb0, g = 0; kb < kb1; kb++, g++) {
                float t[MATS][L];
#pragma unroll
                for (int l = 0; l < L; l++) {
                    t[0][l] = x1[l] * a1;
                    if (GATED) t[MATS - 1][l] = x1[l] * b1;
                    x1[l] = x2[l];
                }
                a1 = a2; b1 = b2;
                fetch(kb + 2, x2, a2, b2);
                const int b = g % S::kBufs;
                if (lane == 0) mbar_wait(tfull(b), (uint32_t)(g / S::kBufs) & 1u, abort_flag, p.status);
                __syncwarp();
                tc_fence_after();
                constexpr int CH = NT < 32 ? NT : 32;                   // columns in registers at a time
#pragma unroll
                for (int m = 0; m < MATS; m++)
#pragma unroll
                    for (int c0 = 0; c0 < NT; c0 += CH) {
                        uint32_t r[CH];
#pragma unroll
                        for (int c = 0; c < CH; c += 16)
                            tmem_ld16(taddr + (uint32_t)((b * MATS + m) * NT + c0 + c), *reinterpret_cast<uint32_t(*)[16]>(&r[c]));
                        tmem_ld_wait();
                        if (m == MATS - 1 && c0 == NT - CH) {           // all of it is in registers: the buffer is free
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(tempty(b));
                        }
#pragma unroll
                        for (int c = 0; c < CH; c++)
                            acc[m][c0 + c] = fmaf(__uint_as_float(r[c]), __shfl_sync(0xffffffffu, t[m][(c0 + c) / 32], (c0 + c) % 32), acc[m][c0 + c]);
                    }
            }
            // every MMA and copy of this CTA is done: the parts go where the stages were, [matrix][row][feature]
            float* part = reinterpret_cast<float*>(gen);
#pragma unroll
            for (int m = 0; m < MATS; m++)
#pragma unroll
                for (int c = 0; c < NT; c++)
                    if (c < nv) part[(m * NT + c) * 128 + tid] = acc[m][c];
        } else if (warp == S::kTmaWarp) {
            if (lane == 0) {
                int g = 0;
                for (int kb = kb0; kb < kb1; kb++, g++) {
                    const int s = g % S::kStages;
                    if (!(early && g < first)) {
                        mbar_wait(empty(s), ((uint32_t)(g / S::kStages) & 1u) ^ 1u, abort_flag, p.status);
                        if (*abort_flag) break;
                        load_weights(kb, s, expert);
                    }
                    tma_load_2d(base + (uint32_t)s * S::kStage + MATS * S::kA, &rows_map, kb * 128, row0, full(s));
                }
                if (*abort_flag)
                    for (int k = max(0, g - S::kStages); k < g; k++) mbar_drain(full(k % S::kStages), (uint32_t)(k / S::kStages) & 1u);
            }
        } else if (lane == 0) {
            const uint32_t idesc = umma_idesc_f16(NT);
            int g = 0;
            for (int kb = kb0; kb < kb1; kb++, g++) {
                const int s = g % S::kStages, b = g % S::kBufs;
                mbar_wait(tempty(b), ((uint32_t)(g / S::kBufs) & 1u) ^ 1u, abort_flag, p.status);
                mbar_wait(full(s), (uint32_t)(g / S::kStages) & 1u, abort_flag, p.status);
                if (*abort_flag) break;
                tc_fence_after();
                const uint32_t at = base + (uint32_t)s * S::kStage;
                const uint64_t rows = umma_desc(at + MATS * S::kA);
#pragma unroll
                for (int m = 0; m < MATS; m++) {
                    const uint64_t w = umma_desc(at + m * S::kA);
#pragma unroll
                    for (int k = 0; k < 4; k++) umma_f8f6f4(tmem + (uint32_t)((b * MATS + m) * NT), w + 2u * k, rows + 2u * k, idesc, k ? 1u : 0u);
                }
                umma_commit(empty(s));
                umma_commit(tfull(b));
            }
            if (*abort_flag && g > 0) mbar_drain(tfull((g - 1) % S::kBufs), (uint32_t)((g - 1) / S::kBufs) & 1u);
        }
        __syncwarp();
        if (split > 1) cluster_sync(); else __syncthreads();
        // ===== join: this CTA's share of the rows, thread = feature ===================================================
        if (warp < 4) {
            const uint32_t mine = base + 4u * tid;
            const int f = f0 + tid;
            for (int c = rank; c < nv; c += split) {
                float v[MATS];
#pragma unroll
                for (int m = 0; m < MATS; m++) {
                    v[m] = 0.f;
                    for (int q = 0; q < split; q++) v[m] += peer_f32(mine + (uint32_t)(m * NT + c) * 512u, (uint32_t)q);
                }
                if (GATED) {
                    const float a = f < p.n ? silu_times(v[0], v[MATS - 1]) : 0.f;
                    uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(a)));
                    uint32_t* t = tops + ((c / split) & 1) * 4;
                    if (lane == 0) t[warp] = top;
                    asm volatile("bar.sync 1, 128;" ::: "memory");
                    top = max(max(t[0], t[1]), max(t[2], t[3]));
                    float scale, lift, factor;
                    f8_act_scale(__uint_as_float(top), scale, lift, factor);
                    const float q = a * lift * factor;
                    if (f < p.n) p.codes[(size_t)(row0 + c) * p.n + f] = (uint8_t)__nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3);
                    if (tid == 0) p.code_scales[(size_t)(f0 / 128) * p.pitch + row0 + c] = scale;
                } else if (f < p.n) {
                    const size_t row = p.route_of_row ? p.route_of_row[row0 + c] : (uint32_t)(row0 + c);
                    p.out[row * p.n + f] = f32_to_bf16_bits(v[0]);
                }
            }
        }
        if (split > 1) cluster_sync();                                   // nobody leaves while its parts are read
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == S::kMmaWarp) tmem_dealloc(tmem, S::kTmem);
}

}  // namespace oco
