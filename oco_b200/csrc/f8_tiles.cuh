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
#include "cluster.cuh"

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
    float* sums;                    // instead of out, where results are summed afterwards: f32 [..][n]
    uint8_t* codes;                 // gated: codes of the activations [row][n]
    float* code_scales;             // and their scales [ceil(n / 128)][pitch]
    uint32_t* status;
    // f8_thin_kernel's other forms: bf16 rows to be rounded (kF8Rows), routes (ids may be null there: dense), the token's sum
    const uint16_t* x;              // bf16 [..][K]
    const uint32_t* ids;            // [tokens][top_k]
    const float* probs;
    const uint16_t* residual;
    int n, K, rows, pitch, top_k, experts;
};

// silu(g) * u. The sigmoid is that of the other formats' tiles, to about 1e-6: of activations that are rounded to four bits
// right away.
__device__ __forceinline__ float silu_times(float g, float u) { return sigmoid_times(g, 1.0f) * g * u; }
// ---- many rows --------------------------------------------------------------------------------------------------------
// PAIR: two SMs multiply one tile of 256 rows (tcgen05.mma.cta_group::2): each brings its own 128 rows and half of the 256
// features, so that an SM fetches 32 KB instead of 48 KB for the same 128 x 256 products of 128 terms.
// Two warpgroups read the accumulators and hold the sums; the third one's warps feed them: TMA, MMA, scales. The 168
// registers a thread starts with are dealt anew, 224 to the sums and 56 to the rest (2 * 224 + 56 = 3 * 168).
template <bool PAIR>
struct F8Wide {
    static constexpr int kRows = PAIR ? 256 : 128;                      // rows of a tile
    static constexpr int kA = 128 * 128, kB = (PAIR ? 128 : 256) * 128, kStage = kA + kB, kStages = PAIR ? 4 : 3;
    static constexpr int kTmaWarp = 8, kMmaWarp = 9, kScaleWarp = 10, kThreads = 384;
    static constexpr int kScaleRun = 4, kScales = 3;                    // scales travel in runs of four blocks, three runs
    static constexpr int kScaleBytes = 128 * 2 * 4;                     // of a block: 128 rows under two blocks of features
    static constexpr int kOutPitch = 256 + 16;                          // a row's 128 results (64 in f32), spread over the banks
    static constexpr int kOut = kStages * kStage, kCtrlAt = kOut + 8 * 32 * kOutPitch;
    static constexpr int kTops = 512, kRing = kTops + 2 * 128 * 4, kCtrl = kRing + kScales * kScaleRun * kScaleBytes;
    static constexpr int kSmem = kCtrlAt + kCtrl + 1024;
    static_assert(kSmem <= 232448, "shared memory of one CTA");
    static_assert(8 * (2 * kStages + 2 + 2 * kScales) + 8 <= kTops, "barriers");
};
template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ float lds_f32(uint32_t at) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void umma_f8f6f4_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// GATED: the 256 columns of a tile are 128 gate and the same 128 up features, the result is silu(gate) * up as codes.
// Launched in clusters of two where PAIR; persistent: CTA (pair) c takes items c, c + CTAs (pairs), ...
template <bool GATED, bool PAIR>
__global__ void __launch_bounds__(F8Wide<PAIR>::kThreads, 1) f8_wide_kernel(const F8TileParams p, const __grid_constant__ CUtensorMap rows_map,
                                                                           const __grid_constant__ CUtensorMap w0_map, const __grid_constant__ CUtensorMap w1_map) {
    using S = F8Wide<PAIR>;
    extern __shared__ unsigned char smem_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = PAIR ? cluster_rank() : 0u;                   // 0: the CTA that issues the MMAs
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t ctrl = base + S::kCtrlAt;
    auto full = [&](int s) { return ctrl + 8u * s; };                   // of the issuing CTA: the stage of both has landed
    auto done = [&](int s) { return ctrl + 8u * (S::kStages + s); };    // the MMAs of the stage: its sums are there, its room is free
    auto tempty = [&](int b) { return ctrl + 8u * (2 * S::kStages + b); };   // of the issuing CTA: both have read
    auto sfull = [&](int q) { return ctrl + 8u * (2 * S::kStages + 2 + q); };
    auto sempty = [&](int q) { return ctrl + 8u * (2 * S::kStages + 2 + S::kScales + q); };
    auto ring = [&](int q, int k) { return ctrl + S::kRing + (uint32_t)(q * S::kScaleRun + k) * S::kScaleBytes; };   // [row][gate, up or first, second block]
    uint32_t* slot = reinterpret_cast<uint32_t*>(gen + S::kCtrlAt + 8 * (2 * S::kStages + 2 + 2 * S::kScales));
    volatile uint32_t* abort_flag = slot + 1;
    uint32_t* tops = reinterpret_cast<uint32_t*>(gen + S::kCtrlAt + S::kTops);   // [2][128]
    const uint32_t lead = PAIR ? map_to_cta(ctrl, 0) : ctrl;
    auto at_lead = [&](uint32_t bar) { return lead + (bar - ctrl); };
    if (tid == 0) {
        for (int s = 0; s < S::kStages; s++) { mbar_init(full(s), 1); mbar_init(done(s), 1); }
        for (int q = 0; q < S::kScales; q++) { mbar_init(sfull(q), 32); mbar_init(sempty(q), 8); }
        for (int b = 0; b < 2; b++) mbar_init(tempty(b), PAIR ? 16 : 8);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == S::kMmaWarp) {
        if (PAIR) { tmem_alloc_pair(smem_u32(slot), 512); tmem_relinquish_pair(); }
        else { tmem_alloc(smem_u32(slot), 512); tmem_relinquish(); }
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync_all();   // both CTAs' barriers exist before anything arrives on them
    tc_fence_after();
    const uint32_t tmem = *slot;
    pdl_wait();                // the kernel before has completed and its writes are visible
    pdl_launch_dependents();

    constexpr int kFeat = GATED ? 128 : 256;
    const int nfeat = (p.n + kFeat - 1) / kFeat, nkb = (p.K + 127) / 128, nfb = (p.n + 127) / 128;
    const int ntiles = p.tiles ? (int)*p.tile_count : (p.rows + S::kRows - 1) / S::kRows;
    const int total = ntiles * nfeat;
    const int first = PAIR ? (int)blockIdx.x >> 1 : (int)blockIdx.x, step = PAIR ? (int)gridDim.x >> 1 : (int)gridDim.x;
    struct Item { int expert, row0, nv, f0; };                          // rows of this CTA's part
    auto item_of = [&](int i) {
        Item r;
        const int t = i / nfeat;
        r.f0 = (i - t * nfeat) * kFeat;
        int end = p.rows;
        r.expert = 0; r.row0 = t * S::kRows;
        if (p.tiles) {
            r.expert = (int)p.tiles[2 * t];
            r.row0 = (int)p.tiles[2 * t + 1];
            end = (int)p.offsets[r.expert + 1];
        }
        r.row0 += 128 * (int)rank;
        r.nv = max(0, min(128, end - r.row0));
        return r;
    };

    if (warp < 8) {
        more_registers<224>();
        // ===== epilogue: thread = row (32 * (warp & 3) + lane), half of the columns (warp >> 2) ====================
        const int erow = (warp & 3) * 32 + lane, half = warp >> 2;
        const uint32_t taddr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t col0 = GATED ? 64u * half : 128u * half, col1 = GATED ? 128u + 64u * half : 128u * half + 64u;
        // results leave through shared memory: a row's part is one bulk copy (a thread's own 16-byte stores would touch
        // 32 rows an instruction, which took as long as the MMAs of an item)
        const uint32_t out_row = base + S::kOut + (uint32_t)(warp * 32 + lane) * S::kOutPitch;
        auto send = [&](void* dst, uint32_t bytes, bool live) {
            fence_proxy_async_smem();
            if (live) asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(out_row), "r"(bytes) : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        };
        auto store16 = [&](int c, const uint32_t (&w)[4]) {
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(out_row + 16u * c), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
        };
        int g = 0, run = 0;
        for (int i = first; i < total; i += step) {
            const Item it = item_of(i);
            uint64_t acc[64];
#pragma unroll
            for (int j = 0; j < 64; j++) acc[j] = 0;
            // scales of a block: gate columns under the gate's, up columns under up's; else under this half's feature block's
            uint64_t t0, t1;
            auto scales = [&](int kb) {
                const int k = kb % S::kScaleRun, q = run % S::kScales;
                if (k == 0) mbar_wait(sfull(q), (uint32_t)(run / S::kScales) & 1u, abort_flag, p.status);
                const uint32_t at = ring(q, k) + 8u * erow;
                const float s0 = lds_f32(at + (GATED ? 0u : 4u * half)), s1 = GATED ? lds_f32(at + 4u) : s0;
                t0 = f32x2(s0, s0);
                t1 = f32x2(s1, s1);
                if (k == S::kScaleRun - 1 || kb == nkb - 1) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(sempty(q));
                    run++;
                }
            };
            scales(0);
            bool there = mbar_try_wait(done(g % S::kStages), (uint32_t)(g / S::kStages) & 1u);
            for (int kb = 0; kb < nkb; kb++, g++) {
                const int b = g & 1, s = g % S::kStages;
                if (!there) mbar_wait(done(s), (uint32_t)(g / S::kStages) & 1u, abort_flag, p.status);
                tc_fence_after();
                const uint32_t at0 = taddr + 256u * b + col0, at1 = taddr + 256u * b + col1;
                uint32_t r[32], u[32];
                auto add = [&](const uint32_t (&v)[32], uint64_t t, int j0) {
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        asm volatile("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc[j0 + j]) : "l"(f32x2_bits(v[2 * j], v[2 * j + 1])), "l"(t));
                };
                tmem_ld32(at0, r);
                tmem_ld32(at0 + 32u, u);
                tmem_ld_wait();
                add(r, t0, 0);
                tmem_ld32(at1, r);                                    // travels while the columns before it are added
                add(u, t0, 16);
                tmem_ld32(at1 + 32u, u);
                tmem_ld_wait();
                tc_fence_before();                                    // all of it is in registers: the buffer is free
                __syncwarp();
                if (lane == 0) {
                    if (PAIR) mbar_arrive_peer(at_lead(tempty(b)));
                    else mbar_arrive(tempty(b));
                }
                const uint64_t last = t1;
                // the next block's scales and a first look at its barrier, under the sums of this one
                if (kb + 1 < nkb) {
                    scales(kb + 1);
                    there = mbar_try_wait(done((g + 1) % S::kStages), (uint32_t)((g + 1) / S::kStages) & 1u);
                }
                add(r, last, 32);
                add(u, last, 48);
            }
            const bool live = erow < it.nv;
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");       // the item before has left its rows
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
                const F8Divider by(__uint_as_float(top));
                const size_t row = (size_t)it.row0 + erow;
                if (live && half == 0) p.code_scales[(size_t)(it.f0 / 128) * p.pitch + row] = by.scale();
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) w[k] = by.codes(acc[8 * c + 2 * k], acc[8 * c + 2 * k + 1]);
                    store16(c, w);
                }
                send(p.codes + row * p.n + f, (uint32_t)max(0, min(64, p.n - f)), live && f < p.n);
            } else {
                const int f = it.f0 + 128 * half;
                const size_t row = !live ? 0 : p.route_of_row ? p.route_of_row[it.row0 + erow] : (uint32_t)(it.row0 + erow);
                if (!PAIR && p.sums) {                                // f32: 64 features at a time
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        if (h) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
#pragma unroll
                        for (int c = 0; c < 16; c++) {
                            float v[4];
                            f32x2_split(acc[32 * h + 2 * c], v[0], v[1]);
                            f32x2_split(acc[32 * h + 2 * c + 1], v[2], v[3]);
                            const uint32_t w[4] = {__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
                            store16(c, w);
                        }
                        const int fh = f + 64 * h;
                        send(p.sums + row * p.n + fh, 4u * (uint32_t)max(0, min(64, p.n - fh)), live && fh < p.n);
                    }
                } else {
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
                        store16(c, w);
                    }
                    send(p.out + row * p.n + f, 2u * (uint32_t)max(0, min(128, p.n - f)), live && f < p.n);
                }
            }
        }
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    } else {
        fewer_registers<56>();
        if (warp == S::kScaleWarp) {
            // ===== scales: four rows a lane times the two blocks of the weights, a run of blocks of K at a time ==========
            int run = 0;
            for (int i = first; i < total; i += step) {
                const Item it = item_of(i);
                const int fb = it.f0 / 128;
                const float* w0 = p.s0 + ((size_t)it.expert * nfb + fb) * nkb;
                const float* w1 = GATED ? p.s1 + ((size_t)it.expert * nfb + fb) * nkb : p.s0 + ((size_t)it.expert * nfb + min(fb + 1, nfb - 1)) * nkb;
                for (int kb = 0; kb < nkb; kb += S::kScaleRun, run++) {
                    const int q = run % S::kScales;
                    float x[S::kScaleRun][4], a[S::kScaleRun], b[S::kScaleRun];
#pragma unroll
                    for (int k = 0; k < S::kScaleRun; k++) {
                        const int at = min(kb + k, nkb - 1);
                        const float* xs = p.row_scales + (size_t)at * p.pitch;
#pragma unroll
                        for (int r = 0; r < 4; r++) x[k][r] = xs[min(it.row0 + lane + 32 * r, p.pitch - 1)];
                        a[k] = w0[at];
                        b[k] = w1[at];
                    }
                    mbar_wait(sempty(q), ((uint32_t)(run / S::kScales) & 1u) ^ 1u, abort_flag, p.status);
#pragma unroll
                    for (int k = 0; k < S::kScaleRun; k++)
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(ring(q, k) + 8u * (lane + 32 * r)), "f"(x[k][r] * a[k]), "f"(x[k][r] * b[k]) : "memory");
                    mbar_arrive(sfull(q));
                }
            }
        } else if (warp == S::kTmaWarp && lane == 0) {
            // ===== operands: this CTA's 128 rows, and its half (PAIR) or all of the features ==============================
            int g = 0;
            for (int i = first; i < total && !*abort_flag; i += step) {
                const Item it = item_of(i);
                const int wrow = it.expert * p.n + it.f0;
                for (int kb = 0; kb < nkb; kb++, g++) {
                    const int s = g % S::kStages;
                    mbar_wait(done(s), ((uint32_t)(g / S::kStages) & 1u) ^ 1u, abort_flag, p.status);
                    if (*abort_flag) break;
                    const uint32_t at = base + (uint32_t)s * S::kStage;
                    if (PAIR) {
                        if (rank == 0) mbar_arrive_expect_tx(full(s), 2 * S::kStage);
                        tma_load_2d_pair(at, &rows_map, kb * 128, it.row0, at_lead(full(s)));
                        if (GATED) tma_load_2d_pair(at + S::kA, rank ? &w1_map : &w0_map, kb * 128, wrow, at_lead(full(s)));
                        else tma_load_2d_pair(at + S::kA, &w0_map, kb * 128, wrow + 128 * (int)rank, at_lead(full(s)));
                    } else {
                        mbar_arrive_expect_tx(full(s), S::kStage);
                        tma_load_2d(at, &rows_map, kb * 128, it.row0, full(s));
                        tma_load_2d(at + S::kA, &w0_map, kb * 128, wrow, full(s));
                        tma_load_2d(at + S::kA + S::kB / 2, GATED ? &w1_map : &w0_map, kb * 128, GATED ? wrow : wrow + 128, full(s));
                    }
                }
            }
        } else if (warp == S::kMmaWarp && rank == 0) {
            // e4m3 x e4m3, f32; M = 128 (256 over the pair), N = 256: columns of this CTA's features, then of the other's.
            // The whole warp waits, one lane issues: what the MMAs of a block cost this warp has to stay below their own time.
            const uint32_t idesc = PAIR ? umma_idesc_f16_pair(256) : umma_idesc_f16(256);
            const uint64_t a0 = umma_desc(base), w0 = umma_desc(base + S::kA);
            const uint32_t d0 = __shfl_sync(0xffffffffu, tmem, 0);
            const int blocks = total > first ? (total - first + step - 1) / step * nkb : 0;
            int s = 0;
            uint32_t turn = 0;                                          // parity of the stages' turn
            for (int g = 0; g < blocks; g++) {
                const int b = g & 1;
                mbar_wait(full(s), turn, abort_flag, p.status);
                mbar_wait(tempty(b), ((uint32_t)(g >> 1) & 1u) ^ 1u, abort_flag, p.status);
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t a = a0 + (uint64_t)(s * (S::kStage >> 4)), w = w0 + (uint64_t)(s * (S::kStage >> 4));
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        if (PAIR) umma_f8f6f4_pair(d0 + 256u * b, a + 2u * k, w + 2u * k, idesc, k ? 1u : 0u);
                        else umma_f8f6f4(d0 + 256u * b, a + 2u * k, w + 2u * k, idesc, k ? 1u : 0u);
                    }
                    if (PAIR) umma_commit_pair(done(s));
                    else umma_commit(done(s));
                }
                __syncwarp();
                if (++s == S::kStages) { s = 0; turn ^= 1u; }
            }
        }
    }
    __syncthreads();
    if (*abort_flag) {
        for (int i = 0; i < 64; i++) __nanosleep(1000);   // let copies and MMAs in flight end before the CTA retires
        __syncthreads();
    }
    tc_fence_before();
    if (PAIR) cluster_sync_all();   // neither CTA retires, or gives its tensor memory back, while the other may still signal or multiply
    else __syncthreads();
    tc_fence_after();
    if (warp == S::kMmaWarp) {
        if (PAIR) tmem_dealloc_pair(tmem, 512);
        else tmem_dealloc(tmem, 512);
    }
}

// ---- few rows ---------------------------------------------------------------------------------------------------------
// What a CTA's rows are:
//   kF8Tiles   codes and scales in memory (f8_rows_kernel, or the gated form of a product before); rows by TMA
//   kF8Rows    bf16 rows, up to 16, that the CTA rounds to codes itself, the blocks of its part of the contraction: no
//              kernel before it. Dense, or one tile per route (one row: the route's token)
//   kF8Concat  one token's routes one behind the other as one long contraction, the weights of the routes in the scales:
//              out = residual + sum_r prob_r (down_r . a_r), no kernel behind it
enum F8Form { kF8Tiles, kF8Rows, kF8Concat };

template <int NT, bool GATED, int FORM>
struct F8Thin {
    static_assert(FORM == kF8Tiles || NT == 16, "the other forms have up to 16 rows");
    static_assert(FORM != kF8Concat || !GATED, "");
    static constexpr int kA = 128 * 128, kMats = GATED ? 2 : 1, kB = FORM == kF8Rows ? 0 : NT * 128, kStage = kMats * kA + kB;
    static constexpr int kCols = FORM == kF8Concat ? 1 : NT;            // columns that are rows
    static constexpr bool kTight = GATED && NT == 64;                   // 128 sums a thread: fewer columns at a time, or one CTA fills an SM's registers
    static constexpr int kBlocks = 8;                                   // kF8Rows: blocks of a CTA's part at most
    static constexpr int kOwn = FORM == kF8Rows ? kBlocks * NT * (128 + 4) : 0;   // their codes, then their scales
    // Shared memory for two CTAs an SM; narrow tiles get by with less, and three or four CTAs hide one another's start and end
    // (64 tokens over 128 experts: 136 -> 114 us).
    static constexpr int kRoom = (NT == 16 && FORM == kF8Tiles ? (GATED ? 70 : 54) : 108) * 1024;
    static constexpr int kStages = (kRoom - kOwn) / kStage > 2 ? (kRoom - kOwn) / kStage : 2;
    static constexpr int kBufs = NT == 16 ? 4 : 2, kTmemUsed = kBufs * kMats * NT;   // narrow tiles: MMAs of more blocks ahead of the sums
    static constexpr int kTmem = kTmemUsed <= 32 ? 32 : kTmemUsed <= 64 ? 64 : kTmemUsed <= 128 ? 128 : 256;
    static constexpr int kTmaWarp = 4, kMmaWarp = 5, kThreads = 192;
    static constexpr int kCtrl = 512;
    static constexpr int kSmem = kStages * kStage + kOwn + kCtrl + 1024;
    static_assert(kMats * kCols * 128 * 4 <= kStages * kStage, "the parts of a split contraction lie where the stages were");
    static_assert(8 * (2 * kStages + 2 * kBufs) + 8 <= 256, "barriers");
};

// One item (a tile of up to NT rows of one expert, 128 features) per cluster; CTA r of its S takes the blocks
// [r * per, ..) of the contraction. x = S * (item), items: feature tile fastest.
//
// Weights travel before the kernel before is waited for: they have been there since they were bound (one row through 4096
// -> 6144 features: 5.8 us, after the wait 6.9), and the tiles and (kF8Concat) the ids come from a kernel that has ended
// when this one may start, since every kernel of a call lets the next one start only after its own wait. kF8Rows with ids
// (a router may just have written them) waits first.
template <int NT, bool GATED, int FORM>
__global__ void __launch_bounds__(F8Thin<NT, GATED, FORM>::kThreads, 2) f8_thin_kernel(const F8TileParams p, const __grid_constant__ CUtensorMap rows_map,
                                                                                   const __grid_constant__ CUtensorMap w0_map,
                                                                                   const __grid_constant__ CUtensorMap w1_map) {
    using S = F8Thin<NT, GATED, FORM>;
    constexpr int MATS = S::kMats, COLS = S::kCols;
    extern __shared__ unsigned char smem_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t own = base + S::kStages * S::kStage, ctrl = own + S::kOwn;
    unsigned char* gctrl = gen + (ctrl - base);
    auto full = [&](int s) { return ctrl + 8u * s; };
    auto empty = [&](int s) { return ctrl + 8u * (S::kStages + s); };
    auto tfull = [&](int b) { return ctrl + 8u * (2 * S::kStages + b); };
    auto tempty = [&](int b) { return ctrl + 8u * (2 * S::kStages + S::kBufs + b); };
    uint32_t* slot = reinterpret_cast<uint32_t*>(gctrl + 8 * (2 * S::kStages + 2 * S::kBufs));
    volatile uint32_t* abort_flag = slot + 1;
    volatile uint32_t* routes = reinterpret_cast<uint32_t*>(gctrl + 256);   // kF8Concat: how many, then (expert, route) of each
    const int split = (int)cluster_size(), rank = (int)cluster_rank();
    const int nfeat = (p.n + 127) / 128, nkb = (p.K + 127) / 128;
    const int item = (int)blockIdx.x / split, tile = item / nfeat, f0 = (item - tile * nfeat) * 128;
    if (tid == 0) {
        for (int s = 0; s < S::kStages; s++) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        for (int b = 0; b < S::kBufs; b++) { mbar_init(tfull(b), 1); mbar_init(tempty(b), 4); }
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (FORM == kF8Concat && warp == 0) {                               // the token's routes that have an expert here
        const uint32_t e = lane < p.top_k ? __ldcg(p.ids + (size_t)tile * p.top_k + lane) : 0xffffffffu;
        const uint32_t live = __ballot_sync(0xffffffffu, e < (uint32_t)p.experts);
        const int at = __popc(live & ((1u << lane) - 1u));
        if ((live >> lane) & 1u) { routes[1 + 2 * at] = e; routes[2 + 2 * at] = lane; }
        if (lane == 0) routes[0] = __popc(live);
    }
    if (warp == S::kMmaWarp) { tmem_alloc(smem_u32(slot), S::kTmem); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    // ---- what this CTA multiplies: rows [row0, row0 + nv) of codes with blocks [q0, q1) of the contraction -----------------
    int expert = 0, row0 = tile * NT, nv = min(NT, p.rows - row0);
    const bool early = FORM != kF8Rows || !p.ids;
    if (FORM == kF8Tiles && p.tiles) {
        if (tile >= (int)__ldcg(p.tile_count)) nv = 0;                  // the whole cluster (read past L1: not waited for yet)
        else {
            expert = (int)__ldcg(p.tiles + 2 * tile);
            row0 = (int)__ldcg(p.tiles + 2 * tile + 1);
            nv = min(NT, (int)__ldcg(p.offsets + expert + 1) - row0);
        }
    }
    if (FORM == kF8Concat) nv = 1;
    if (!early) {
        pdl_wait();            // the kernel before has completed and its writes are visible
        pdl_launch_dependents();
        const uint32_t e = p.ids[tile];                                 // a tile per route, its row
        row0 = tile;
        nv = e < (uint32_t)p.experts ? 1 : 0;
        expert = nv ? (int)e : 0;
    }
    const int blocks = FORM == kF8Concat ? (int)routes[0] * nkb : nkb, per = (blocks + split - 1) / split;
    const int q0 = min(blocks, rank * per), q1 = nv > 0 ? min(blocks, q0 + per) : q0;
    auto load_weights = [&](int q, int s) {
        const uint32_t at = base + (uint32_t)s * S::kStage;
        int e = expert, kb = q;
        if (FORM == kF8Concat) { const int r = q / nkb; kb = q - r * nkb; e = (int)routes[1 + 2 * r]; }
        mbar_arrive_expect_tx(full(s), S::kStage);
        tma_load_2d(at, &w0_map, kb * 128, e * p.n + f0, full(s));
        if (GATED) tma_load_2d(at + S::kA, &w1_map, kb * 128, e * p.n + f0, full(s));
    };
    const int first = min(S::kStages, q1 - q0);                         // stages filled before anything is waited for
    if (warp == S::kTmaWarp && lane == 0)
        for (int k = 0; k < first; k++) load_weights(q0 + k, k);
    if (early) {
        pdl_wait();
        pdl_launch_dependents();
    }
    if (nv > 0) {
        if (warp < 4) {
            if (FORM == kF8Rows) {
                // ===== rows to codes: half a warp per row and block (the swizzled layout that TMA would have written) =======
                const int hl = lane & 15, nb = q1 - q0, units = nv * nb;
                auto fetch = [&](int u) {
                    if (u >= units) return make_uint4(0, 0, 0, 0);
                    const int c = u / nb, k = (q0 + u - c * nb) * 128 + 8 * hl;
                    const size_t row = p.ids ? (size_t)(tile / p.top_k) : (size_t)(row0 + c);
                    return k < p.K ? *reinterpret_cast<const uint4*>(p.x + row * p.K + k) : make_uint4(0, 0, 0, 0);
                };
                uint4 next = fetch(tid >> 4);
                for (int both = 2 * warp; both < units; both += 8) {   // all lanes of the warp stay together
                    const int u = both + (lane >> 4);
                    const uint4 v[1] = {next};
                    next = fetch(u + 8);
                    uint2 code[1];
                    float scale[1];
                    f8_blocks(v, code, scale);
                    if (u >= units) continue;
                    const int c = u / nb, i = u - c * nb;
                    const uint32_t at = own + (uint32_t)(i * NT * 128 + (c >> 3) * 1024 + (c & 7) * 128) + ((((uint32_t)hl >> 1) ^ (uint32_t)(c & 7)) << 4) + 8u * (hl & 1);
                    asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(at), "r"(code[0].x), "r"(code[0].y) : "memory");
                    if (hl == 0) reinterpret_cast<float*>(gen + (own - base) + S::kBlocks * NT * 128)[i * NT + c] = scale[0];
                }
                fence_proxy_async_smem();
                asm volatile("bar.sync 2, 160;" ::: "memory");          // with the MMA warp
            }
            // ===== thread = feature, columns = rows ===============================================================
            const uint32_t taddr = tmem + ((uint32_t)(warp * 32) << 16);
            constexpr int L = (NT + 31) / 32;                           // row scales a lane holds
            float acc[MATS][COLS], x1[L], x2[L], a1 = 0.f, a2 = 0.f, b1 = 0.f, b2 = 0.f;
#pragma unroll
            for (int m = 0; m < MATS; m++)
#pragma unroll
                for (int c = 0; c < COLS; c++) acc[m][c] = 0.f;
            auto fetch = [&](int q, float (&x)[L], float& a, float& b) {
                if (q >= q1) return;
                int kb = q, e = expert;
                if (FORM == kF8Concat) {
                    const int r = q / nkb;
                    kb = q - r * nkb;
                    e = (int)routes[1 + 2 * r];
                    const size_t row = (size_t)tile * p.top_k + routes[2 + 2 * r];
                    x[0] = p.row_scales[(size_t)kb * p.pitch + row] * p.probs[row];
                } else if (FORM == kF8Rows) {
                    x[0] = reinterpret_cast<const float*>(gen + (own - base) + S::kBlocks * NT * 128)[(q - q0) * NT + lane % NT];
                } else {
#pragma unroll
                    for (int l = 0; l < L; l++) x[l] = p.row_scales[(size_t)kb * p.pitch + min(row0 + 32 * l + (NT < 32 ? lane % NT : lane), p.pitch - 1)];
                }
                const size_t at = ((size_t)e * nfeat + f0 / 128) * nkb + kb;
                a = p.s0[at];
                if (GATED) b = p.s1[at];
            };
            fetch(q0, x1, a1, b1);
            fetch(q0 + 1, x2, a2, b2);
            for (int q = q0, g = 0; q < q1; q++, g++) {
                float t[MATS][L];
#pragma unroll
                for (int l = 0; l < L; l++) {
                    t[0][l] = x1[l] * a1;
                    if (GATED) t[MATS - 1][l] = x1[l] * b1;
                    x1[l] = x2[l];
                }
                a1 = a2; b1 = b2;
                fetch(q + 2, x2, a2, b2);
                const int b = g % S::kBufs;
                mbar_wait(tfull(b), (uint32_t)(g / S::kBufs) & 1u, abort_flag, p.status);
                __syncwarp();
                tc_fence_after();
                constexpr int CH = NT < 32 || S::kTight ? 16 : 32;      // columns in registers at a time
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
                        if (FORM == kF8Concat) acc[0][0] = fmaf(__uint_as_float(r[0]), t[0][0], acc[0][0]);
                        else {
#pragma unroll
                            for (int c = 0; c < CH; c++)
                                if (c0 + c < COLS) acc[m][(c0 + c) % COLS] = fmaf(__uint_as_float(r[c]), __shfl_sync(0xffffffffu, t[m][(c0 + c) / 32], (c0 + c) % 32), acc[m][(c0 + c) % COLS]);
                        }
                    }
            }
            // every MMA and copy of this CTA is done: the parts go where the stages were, [matrix][row][feature]
            float* part = reinterpret_cast<float*>(gen);
#pragma unroll
            for (int m = 0; m < MATS; m++)
#pragma unroll
                for (int c = 0; c < COLS; c++)
                    if (c < nv) part[(m * COLS + c) * 128 + tid] = acc[m][c];
        } else if (warp == S::kTmaWarp) {
            if (lane == 0) {
                int g = 0;
                for (int q = q0; q < q1; q++, g++) {
                    const int s = g % S::kStages;
                    if (g >= first) {
                        mbar_wait(empty(s), ((uint32_t)(g / S::kStages) & 1u) ^ 1u, abort_flag, p.status);
                        if (*abort_flag) break;
                        load_weights(q, s);
                    }
                    if (FORM == kF8Tiles) tma_load_2d(base + (uint32_t)s * S::kStage + MATS * S::kA, &rows_map, q * 128, row0, full(s));
                    if (FORM == kF8Concat) {
                        const int r = q / nkb;
                        tma_load_2d(base + (uint32_t)s * S::kStage + S::kA, &rows_map, (q - r * nkb) * 128, tile * p.top_k + (int)routes[2 + 2 * r], full(s));
                    }
                }
                if (*abort_flag)
                    for (int k = max(0, g - S::kStages); k < g; k++) mbar_drain(full(k % S::kStages), (uint32_t)(k / S::kStages) & 1u);
            }
        } else {
            if (FORM == kF8Rows) asm volatile("bar.sync 2, 160;" ::: "memory");
            const uint32_t idesc = umma_idesc_f16(NT), d0 = __shfl_sync(0xffffffffu, tmem, 0);
            int g = 0;
            for (int q = q0; q < q1; q++, g++) {
                const int s = g % S::kStages, b = g % S::kBufs;
                mbar_wait(tempty(b), ((uint32_t)(g / S::kBufs) & 1u) ^ 1u, abort_flag, p.status);
                mbar_wait(full(s), (uint32_t)(g / S::kStages) & 1u, abort_flag, p.status);
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t at = base + (uint32_t)s * S::kStage;
                    const uint64_t rows = umma_desc(FORM == kF8Rows ? own + (uint32_t)(q - q0) * NT * 128 : at + MATS * S::kA);
#pragma unroll
                    for (int m = 0; m < MATS; m++) {
                        const uint64_t w = umma_desc(at + m * S::kA);
#pragma unroll
                        for (int k = 0; k < 4; k++) umma_f8f6f4(d0 + (uint32_t)((b * MATS + m) * NT), w + 2u * k, rows + 2u * k, idesc, k ? 1u : 0u);
                    }
                    umma_commit(empty(s));
                    umma_commit(tfull(b));
                }
                __syncwarp();
            }
            if (*abort_flag && g > 0) mbar_drain(tfull((g - 1) % S::kBufs), (uint32_t)((g - 1) / S::kBufs) & 1u);
        }
        __syncwarp();
        if (split > 1) cluster_sync_all(); else __syncthreads();
        // ===== join: this CTA's share of the rows, a warp per row, four features a lane ================================
        const int f = f0 + 4 * lane;
        for (int c = rank + split * warp; c < nv; c += split * (S::kThreads / 32)) {
            float4 v[MATS];
#pragma unroll
            for (int m = 0; m < MATS; m++) {
                const uint32_t at = base + (uint32_t)(m * COLS + c) * 512u + 16u * lane;
                v[m] = peer_f32x4(at, 0);
#pragma unroll 4
                for (int q = 1; q < split; q++) {
                    const float4 w = peer_f32x4(at, (uint32_t)q);
                    v[m].x += w.x; v[m].y += w.y; v[m].z += w.z; v[m].w += w.w;
                }
            }
            if (GATED) {
                const bool in = f < p.n;                                // n is a multiple of 32
                const float4 u = v[MATS - 1];
                const float a[4] = {in ? silu_times(v[0].x, u.x) : 0.f, in ? silu_times(v[0].y, u.y) : 0.f, in ? silu_times(v[0].z, u.z) : 0.f,
                                    in ? silu_times(v[0].w, u.w) : 0.f};
                const uint32_t top = __reduce_max_sync(0xffffffffu, max(max(__float_as_uint(fabsf(a[0])), __float_as_uint(fabsf(a[1]))),
                                                                        max(__float_as_uint(fabsf(a[2])), __float_as_uint(fabsf(a[3])))));
                const F8Divider by(__uint_as_float(top));
                if (in) *reinterpret_cast<uint32_t*>(p.codes + (size_t)(row0 + c) * p.n + f) = by.codes(f32x2(a[0], a[1]), f32x2(a[2], a[3]));
                if (lane == 0) p.code_scales[(size_t)(f0 / 128) * p.pitch + row0 + c] = by.scale();
            } else if (f < p.n) {
                size_t row = FORM == kF8Concat ? (size_t)tile : (size_t)(row0 + c);
                if (FORM == kF8Tiles && p.route_of_row) row = p.route_of_row[row0 + c];
                if (FORM == kF8Concat) {
                    const uint2 q = *reinterpret_cast<const uint2*>(p.residual + row * p.n + f);
                    v[0].x += __uint_as_float(q.x << 16); v[0].y += __uint_as_float(q.x & 0xffff0000u);
                    v[0].z += __uint_as_float(q.y << 16); v[0].w += __uint_as_float(q.y & 0xffff0000u);
                }
                if (FORM == kF8Tiles && p.sums) {
                    *reinterpret_cast<float4*>(p.sums + row * p.n + f) = v[0];
                    continue;
                }
                const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0].x, v[0].y), hi = __floats2bfloat162_rn(v[0].z, v[0].w);
                *reinterpret_cast<uint2*>(p.out + row * p.n + f) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
            }
        }
        if (split > 1) cluster_sync_all();                                   // nobody leaves while its parts are read
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == S::kMmaWarp) tmem_dealloc(tmem, S::kTmem);
}

}  // namespace oco
