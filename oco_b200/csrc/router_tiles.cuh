// The router product on the tensor cores: logits[t][e] = sum_k x[t][k] w[e][k] to the accuracy of f32 sums.
//
// The rows are bf16; an f32 weight is the exact sum of three bf16 pieces of falling size (8 bits of its 24 each), laid
// out once when the weights are bound. Three kind::f16 products with bf16 operands then add exact terms into f32
// accumulators. What is left is the rounding of the sums, which tensor memory cuts off instead of rounding to nearest:
// an MMA adds 16 products and the accumulator, each cut at 2^-25 of the largest one's power of two, and cuts the sum to
// 24 bits (seen on single terms of falling size beside one of size 1). So the largest pieces have an accumulator of their
// own, and after every 64 terms (four additions to it) both are read out and added, rounding to nearest, to sums in
// registers.
//
// The selection has to know how far a logit may be off. In units of 2^-24 |x| |w|: 17 / 2 + 2 for each MMA that a term is
// in its accumulator for: four for those of the first, one for those of the last. So norms are taken of every fourth 16
// columns. 2^-8 of eight MMAs for the smaller pieces and one unit for the sum of both accumulators: one and a half. The
// sums in registers and of the parts: 2^-24 of the largest partial sum of a row, which is kept, for each addition. The
// rows' norms are taken from the tiles in shared memory by the warps that wait for the MMAs anyway.
//
// One item = 128 rows x 128 experts; a contraction is split over the CTAs of a cluster while items do not fill the SMs,
// and the parts are added through distributed shared memory in the order of their ranks. Each stage of shared memory
// holds 64 columns of the rows and of the three pieces (64 KB). All waits are bounded (mbar_wait).
#pragma once
#include "cluster.cuh"
#include "select.cuh"

namespace oco {

struct RouterTile {
    static constexpr int kTile = 128 * 128, kStage = 4 * kTile, kStages = 3;
    static constexpr int kPitch = 132;                   // f32 of a row of the parts: eight rows' 16-byte pieces fill the banks
    static constexpr int kRowsAt = 128 * kPitch;         // behind the parts: [row][4 sums of squares, the largest sums of both halves, -, -]
    static constexpr int kTmaWarp = 8, kMmaWarp = 9, kThreads = 320;   // warps 0 .. 7 hold the sums
    static constexpr int kCtrl = 256, kSmem = kStages * kStage + kCtrl + 1024;
    static_assert((kRowsAt + 128 * 8) * 4 <= kStages * kStage, "the parts lie where the stages were");
};

// Weights -> three bf16 pieces [piece][Ep][H], Ep = experts rounded up to 128 (rows behind the last expert are zero).
__global__ void __launch_bounds__(256) router_pieces_kernel(const float* __restrict__ w, uint16_t* __restrict__ pieces, int E, int Ep, int H) {
    const size_t n = (size_t)Ep * H;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const float v = i < (size_t)E * H ? w[i] : 0.0f;
        const float a = bf16_round(v);
        const bool whole = !nonfinite(a);                // an infinite or NaN weight stands in its first piece alone
        const float b = whole ? bf16_round(v - a) : 0.0f, c = whole ? v - a - b : 0.0f;
        pieces[i] = f32_to_bf16_bits(a);
        pieces[n + i] = f32_to_bf16_bits(b);
        pieces[2 * n + i] = f32_to_bf16_bits(c);
    }
}

// The largest Euclidean norms of an expert's weights (SelectParams::w_norm), rounded up (`largest`: zero before). An expert
// with a weight that is not finite has no finite logit.
__global__ void __launch_bounds__(256) router_norms_kernel(const float* __restrict__ w, uint32_t* __restrict__ largest, int H) {
    __shared__ double part[16];
    double s = 0.0;
    for (int k = threadIdx.x; k < H; k += 256) {           // a thread stays with its fourth
        const double v = (double)w[(size_t)blockIdx.x * H + k];
        s = fma(v, v, s);
    }
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if ((threadIdx.x & 15) == 0) part[threadIdx.x >> 4] = s;
    __syncthreads();
    if (threadIdx.x >= 5) return;
    s = 0.0;
    for (int i = 0; i < 16; i++)
        if (threadIdx.x == 4 || i % 4 == (int)threadIdx.x) s += part[i];
    if (s < INFINITY) atomicMax(largest + threadIdx.x, __float_as_uint(__double2float_ru(sqrt(s))));
}

__global__ void __launch_bounds__(RouterTile::kThreads, 1) router_tile_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map,
                                                                             float* __restrict__ logits, float* __restrict__ errors, const float* __restrict__ w_norm,
                                                                             int rows, int E, int Ep, int H, uint32_t* status) {
    using S = RouterTile;
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
    const int split = (int)cluster_size(), rank = (int)cluster_rank();
    const int chunks = (H + 63) / 64, per = (chunks + split - 1) / split, c0 = min(chunks, rank * per), c1 = min(chunks, c0 + per);
    const int etiles = Ep / 128, item = (int)blockIdx.x / split, row0 = item / etiles * 128, e0 = item % etiles * 128;
    if (tid == 0) {
        for (int s = 0; s < S::kStages; s++) { mbar_init(full(s), 1); mbar_init(empty(s), 9); }   // the MMAs, and the warps that read the rows
        for (int b = 0; b < 2; b++) { mbar_init(tfull(b), 1); mbar_init(tempty(b), 8); }
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == S::kMmaWarp) { tmem_alloc(smem_u32(slot), 512); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    auto load_pieces = [&](int c, int s) {
        const uint32_t at = base + (uint32_t)s * S::kStage;
        mbar_arrive_expect_tx(full(s), S::kStage);
#pragma unroll
        for (int q = 0; q < 3; q++) tma_load_2d(at + (1 + q) * S::kTile, &w_map, c * 64, q * Ep + e0, full(s));
    };
    // the pieces were laid out when the weights were bound: their first tiles travel while the kernel before still runs
    const int first = min(S::kStages, c1 - c0);
    if (warp == S::kTmaWarp && lane == 0)
        for (int k = 0; k < first; k++) load_pieces(c0 + k, k);
    pdl_wait();                // the kernel before has completed and its writes are visible
    pdl_launch_dependents();

    float* part = reinterpret_cast<float*>(gen);
    if (warp < 8) {
        // thread = row 32 * (warp & 3) + lane, half of the columns
        const int row = (warp & 3) * 32 + lane, col0 = warp < 4 ? 0 : 64;
        uint64_t sum[32];
        float big = 0.f;                                                   // largest magnitude of a partial sum
        uint64_t squares[2] = {0, 0};                                      // of half of the row's elements, in two of the four parts
        uint32_t some = 0;
#pragma unroll
        for (int j = 0; j < 32; j++) sum[j] = 0;
        const uint32_t taddr = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)col0;
        for (int c = c0, g = 0; c < c1; c++, g++) {
            const int s = g % S::kStages, b = g & 1;
            mbar_wait(full(s), (uint32_t)(g / S::kStages) & 1u, abort_flag, status);
            const unsigned char* mine = gen + s * S::kStage + row * 128;
#pragma unroll
            for (int j = 0; j < 4; j++) {                                  // in an order that keeps eight rows on different banks
                const uint4 q = *reinterpret_cast<const uint4*>(mine + (((j + (warp & 4)) ^ (row & 7)) << 4));
                const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint64_t v = f32x2_bits(w[k] << 16, w[k] & 0xffff0000u);
                    squares[j / 2] = fma_f32x2(v, v, squares[j / 2]);
                }
                some |= q.x | q.y | q.z | q.w;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty(s));
            mbar_wait(tfull(b), (uint32_t)(g >> 1) & 1u, abort_flag, status);
            tc_fence_after();
            const uint32_t at = taddr + 256u * b;
            uint32_t r[2][16], u[2][16];
            tmem_ld16(at, r[0]);
            tmem_ld16(at + 128u, u[0]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                tmem_ld_wait();
                if (i < 3) {                                               // the next columns travel while these are added
                    tmem_ld16(at + 16u * (i + 1), r[(i + 1) & 1]);
                    tmem_ld16(at + 16u * (i + 1) + 128u, u[(i + 1) & 1]);
                } else {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(tempty(b));
                }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    uint64_t both;                                         // volatile: not before the wait above
                    asm volatile("add.rn.f32x2 %0, %1, %2;" : "=l"(both) : "l"(f32x2_bits(r[i & 1][2 * j], r[i & 1][2 * j + 1])),
                                 "l"(f32x2_bits(u[i & 1][2 * j], u[i & 1][2 * j + 1])));
                    uint64_t& t = sum[8 * i + j];
                    t = add_f32x2(t, both);
                    float lo, hi;
                    f32x2_split(t, lo, hi);
                    big = fmaxf(big, fmaxf(fabsf(lo), fabsf(hi)));
                }
            }
        }
        // every MMA of this CTA is done, and the rows have been read: the parts go where the stages were
        asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll
        for (int j = 0; j < 32; j += 2) *reinterpret_cast<ulonglong2*>(part + row * S::kPitch + col0 + 2 * j) = make_ulonglong2(sum[j], sum[j + 1]);
        float* of_row = part + S::kRowsAt + row * 8;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            float even, odd;
            f32x2_split(squares[i], even, odd);
            of_row[2 * (warp >> 2) + i] = even + odd + (some & 0x7fff7fffu ? kLostSquares : 0.f);
        }
        of_row[4 + (warp >> 2)] = big;
    } else if (warp == S::kTmaWarp) {
        if (lane == 0) {
            int g = 0;
            for (int c = c0; c < c1; c++, g++) {
                const int s = g % S::kStages;
                if (g >= first) {
                    mbar_wait(empty(s), ((uint32_t)(g / S::kStages) & 1u) ^ 1u, abort_flag, status);
                    if (*abort_flag) break;
                    load_pieces(c, s);
                }
                tma_load_2d(base + (uint32_t)s * S::kStage, &x_map, c * 64, row0, full(s));
            }
            if (*abort_flag)
                for (int k = max(0, g - S::kStages); k < g; k++) mbar_drain(full(k % S::kStages), (uint32_t)(k / S::kStages) & 1u);
        }
    } else {
        const uint32_t idesc = umma_idesc_f16(128) | (1u << 7) | (1u << 10);       // both operands bf16
        const uint32_t d0 = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t x0 = umma_desc(base), w0 = umma_desc(base + S::kTile);
        for (int c = c0, g = 0; c < c1; c++, g++) {
            const int s = g % S::kStages, b = g & 1;
            mbar_wait(tempty(b), ((uint32_t)(g >> 1) & 1u) ^ 1u, abort_flag, status);
            mbar_wait(full(s), (uint32_t)(g / S::kStages) & 1u, abort_flag, status);
            tc_fence_after();
            if (elect_one()) {
                const uint64_t at = (uint64_t)(s * (S::kStage >> 4));
#pragma unroll
                for (int q = 0; q < 3; q++)
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        umma_f16(d0 + 256u * b + (q ? 128u : 0u), x0 + at + 2u * k, w0 + at + (uint64_t)(q * (S::kTile >> 4)) + 2u * k, idesc,
                                 q < 2 && k == 0 ? 0u : 1u);
                umma_commit(empty(s));
                umma_commit(tfull(b));
            }
            __syncwarp();
        }
    }
    __syncthreads();
    if (*abort_flag) {
        for (int i = 0; i < 64; i++) __nanosleep(1000);   // let copies and MMAs in flight end before the CTA goes on
        __syncthreads();
    }
    if (split > 1) cluster_sync_all();
    // join: this CTA's share of the rows, a warp per row, four experts a lane
    const int live = min(128, rows - row0), cols = min(128, E - e0), c = 4 * lane;
    const bool wide = (E & 3) == 0 && ((uintptr_t)logits & 15u) == 0;
    if (tid < live && tid % split == rank) {                               // how far the row's logits may be off
        float n[4] = {0.f, 0.f, 0.f, 0.f}, big0 = 0.f, big1 = 0.f;
#pragma unroll
        for (int q = 0; q < 8; q++) {                                      // all on their way at once
            if (q >= split) continue;
            const uint32_t at = base + 4u * (uint32_t)(S::kRowsAt + tid * 8);
            const float4 squares = peer_f32x4(at, (uint32_t)q), largest = peer_f32x4(at + 16u, (uint32_t)q);
            n[0] += squares.x; n[1] += squares.y; n[2] += squares.z; n[3] += squares.w;
            big0 += largest.x; big1 += largest.y;
        }
        float e = product_error(1.5f, n[0] + n[1] + n[2] + n[3], w_norm[4]) + 1.01f * 5.9604645e-8f * (float)(per + split) * fmaxf(big0, big1);
#pragma unroll
        for (int i = 0; i < 4; i++) e += product_error(10.6f * (float)(4 - i), n[i], w_norm[i]);
        errors[(size_t)(e0 / 128) * rows + row0 + tid] = e;
    }
    for (int r = rank + split * warp; r < live; r += split * (S::kThreads / 32)) {
        const uint32_t at = base + 4u * (uint32_t)(r * S::kPitch + c);
        float4 v = peer_f32x4(at, 0);
#pragma unroll 7
        for (int q = 1; q < split; q++) {
            const float4 w = peer_f32x4(at, (uint32_t)q);
            v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
        }
        float* dst = logits + (size_t)(row0 + r) * E + e0 + c;
        if (wide && c < cols) *reinterpret_cast<float4*>(dst) = v;
        else {
            if (c < cols) dst[0] = v.x;
            if (c + 1 < cols) dst[1] = v.y;
            if (c + 2 < cols) dst[2] = v.z;
            if (c + 3 < cols) dst[3] = v.w;
        }
    }
    tc_fence_before();
    if (split > 1) cluster_sync_all();                   // nobody leaves while its parts are read
    else __syncthreads();
    tc_fence_after();
    if (warp == S::kMmaWarp) tmem_dealloc(tmem, 512);
}

}  // namespace oco
