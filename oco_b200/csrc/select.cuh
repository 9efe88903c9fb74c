// Selection of a token's experts from its logits, with groups of experts, for one warp per token.
//
// Lane l owns the VPL consecutive experts l * VPL .. l * VPL + VPL - 1, so that the lowest lane, and within it the lowest
// element, is the lowest expert index: equal values go to the lower index without a comparison of indices.
//
// Everything is first done in 32 bits. Two ranking values that lie within each other's error (rounding of the score, of
// score + bias, and the error of the logit where it came from the router product) leave their order open; such a token
// is settled in 64 bits, where the logits that matter are summed again from x and the weights. With continuous logits that
// is a token in a few hundred where logits are given or rows are few, one in thirty behind the tensor cores, whose sums
// have the wider bound.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace oco {

constexpr int kSelMaxExperts = 512, kSelMaxTopK = 16, kSelMaxGroups = 32;

struct SelectParams {
    const float* logits;     // [rows, E]
    const float* bias;       // [E] or null
    const uint16_t* x;       // rows the logits were made of, bf16 [rows, H]; null: the logits are exact as given
    const float* w;          // f32 [E, H]
    uint32_t* ids;
    float* probs;
    uint32_t* status;        // null, or a status word: set = nothing is written
    const float* errors;     // behind the product: largest error of a row's logits, [tiles of 128 experts][rows]
    const float* w_norm;     // largest Euclidean norms of an expert's weights: of every fourth 16 columns from 0, 16, 32, 48 on, and of all
    int rows, E, H, K, G, TG, best, score, normalize;
    float scale;
};

// Monotone map of a float to an unsigned key: larger value, larger key. NaN ranks below everything (key 1); 0 is left
// for "not a candidate".
__device__ __forceinline__ uint32_t rank_key(float f) {
    const uint32_t u = __float_as_uint(f + 0.0f);                  // -0 becomes +0: they are equal
    const uint32_t k = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
    return f != f ? 1u : max(k, 2u);
}
__device__ __forceinline__ float key_rank(uint32_t k) {
    return __uint_as_float(k ^ (k & 0x80000000u ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ float warp_sum_f(float v) {
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// Error of a logit that a product of 32-bit sums has made. Its partial sums are as large as the terms make them, however
// small the logit is where large terms cancel, so the bound is one on sums of |x w|: roundings of 2^-24 each (`units` of
// them at most on the way of a term) times |x| |w| (Euclidean norms: no smaller than the sum of |x w|). Where the sum of
// squares overflows nothing is known of the logits. 1.01: the rounding of all this. kLostSquares: what squares below 2^-126
// may have lost in a row of 16384; rows of zeros go without, their logits are exact.
constexpr float kLostSquares = 2e-34f;
__device__ __forceinline__ float product_error(float units, float squares, float w_norm) {
    const float e = 1.01f * units * 5.9604645e-8f * w_norm * sqrtf(squares);
    return e < 1e30f ? e : INFINITY;
}
// A sigmoid in 32 bits: s (1 - s) 2^-22 from the exponential's two units in the last place, the sum's rounding and the
// quotient's two units: below 4e-7.
// A softmax score relative to the largest one: the same and the rounding of l - top (x e^-x < 0.37), the sum and its
// reciprocal. kHalfUlp: the rounding of score + bias.
// kFarError: up to here e^d - 1 is d but for a twentieth. kLeast: 2^-126, below which the last bits of a value (an index
// stands there in a sorted key) weigh more than its size tells.
constexpr float kSigmoidError = 4e-7f, kScoreError = 6e-7f, kHalfUlp = 6e-8f, kFarError = 0.01f, kLeast = 1.1754944e-38f;

// ---- exact logits ----------------------------------------------------------------------------------------------------
// Partial sums of two experts' logits in 64 bits: thread t of T takes the columns 4 t .. 4 t + 3 of every 4 T.
__device__ __forceinline__ void exact_parts(const SelectParams& p, int row, int t, int T, int a, int b, double& la, double& lb) {
    const float4* wa = reinterpret_cast<const float4*>(p.w + (size_t)a * p.H);
    const float4* wb = reinterpret_cast<const float4*>(p.w + (size_t)b * p.H);
    const uint2* xr = reinterpret_cast<const uint2*>(p.x + (size_t)row * p.H);
    double a0 = 0, a1 = 0, b0 = 0, b1 = 0;
#pragma unroll 4
    for (int k = t; k < p.H / 4; k += T) {
        const float4 u = __ldg(wa + k), v = __ldg(wb + k);
        const uint2 q = xr[k];
        const double x0 = (double)__uint_as_float(q.x << 16), x1 = (double)__uint_as_float(q.x & 0xffff0000u);
        const double x2 = (double)__uint_as_float(q.y << 16), x3 = (double)__uint_as_float(q.y & 0xffff0000u);
        a0 = fma((double)u.x, x0, a0); a1 = fma((double)u.y, x1, a1); a0 = fma((double)u.z, x2, a0); a1 = fma((double)u.w, x3, a1);
        b0 = fma((double)v.x, x0, b0); b1 = fma((double)v.y, x1, b1); b0 = fma((double)v.z, x2, b0); b1 = fma((double)v.w, x3, b1);
    }
    la = warp_sum_d(a0 + a1);
    lb = warp_sum_d(b0 + b1);
}
// By one warp: 6 us for 4096 columns, most of it the way of the loads.
__device__ __noinline__ void exact_logits(const SelectParams& p, int row, int lane, int a, int b, double& la, double& lb) { exact_parts(p, row, lane, 32, a, b, la, lb); }

// By the eight warps of a CTA, for all of its open rows together: an eighth of every sum each.
struct SelectShared {
    int row[8], count[8];        // of each warp: its row, and how many logits it wants
    int want[8][32];             // of which experts
    double part[8][8][32];       // [warp that summed][warp that wants][place]
};
__device__ __noinline__ void exact_wanted(const SelectParams& p, SelectShared& sh) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int w = 0; w < 8; w++)
        for (int i = 0, n = sh.count[w]; i < n; i += 2) {
            const int j = min(i + 1, n - 1);
            double la, lb;
            exact_parts(p, sh.row[w], threadIdx.x, 256, sh.want[w][i], sh.want[w][j], la, lb);
            if (lane == 0) { sh.part[warp][w][i] = la; sh.part[warp][w][j] = lb; }
        }
    __syncthreads();
}

// ---- 64-bit path ---------------------------------------------------------------------------------------------------
struct Best { double v; int i; };
// The largest value of the warp, of the lowest lane among equals; i = -1: no candidate. Two reductions over the halves of
// a key that is ordered as the value is (a tree of exchanges of doubles takes three times as long).
__device__ __forceinline__ Best warp_best(Best b) {
    const long long u = __double_as_longlong(b.v + 0.0);
    const unsigned long long k = (unsigned long long)(u ^ (u >> 63)) ^ (u < 0 ? 0ull : 0x8000000000000000ull);
    const bool in = b.i >= 0;
    const uint32_t hi = warp_max(in ? (uint32_t)(k >> 32) : 0u);
    const bool first = in && (uint32_t)(k >> 32) == hi;
    const uint32_t lo = warp_max(first ? (uint32_t)k : 0u), lanes = __ballot_sync(0xffffffffu, first && (uint32_t)k == lo);
    if (!lanes) return Best{0.0, -1};
    const int from = __ffs((int)lanes) - 1;
    return Best{__shfl_sync(0xffffffffu, b.v, from), __shfl_sync(0xffffffffu, b.i, from)};
}

// One token in 64 bits, by a warp. `l`: the lane's logits, `precise`: bit i: element i's is exact, `d`: the largest error of
// the others (0: none). Every value is held with its error, and what is decided between two values is settled when their
// intervals do not overlap. Returns the lane's elements whose exact logits could turn a decision; none in the whole warp:
// ids and weights are written. Ranked is score + bias, without a bias the logit itself: scores that have run into 0 or 1
// keep the order of their logits. Not inlined: it is rare and would cost the 32-bit path registers.
template <int VPL>
__device__ __noinline__ uint32_t exact_step(const SelectParams& p, int row, int lane, double d, const double (&l)[VPL], uint32_t precise) {
    const int E = p.E, gs = p.E / p.G;
    const bool soft = p.score == OCO_SCORE_SOFTMAX, two = p.best == 2 && gs > 1;
    const bool scored = !p.bias && two;                                // groups are worth scores, experts are ranked by logits
    const bool far = d > 0.5;                                          // up to here e^d - 1 is below d (1 + d); scores lie in 0 .. 1 in any case
    double s[VPL], r[VPL], er[VPL], w[VPL], ew[VPL];                   // score, rank and part of a group's worth with their errors
    double top = -1.0 / 0.0, z = 0.0;
    uint32_t in = 0;                                                   // bit i: an expert that can be chosen
    bool all = true;
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        if (lane * VPL + i >= E) continue;
        in |= 1u << i;
        top = fmax(top, l[i]);
        all = all && ((precise >> i) & 1u);
    }
#pragma unroll
    for (int k = 16; k >= 1; k >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, k));
    all = __all_sync(0xffffffffu, all);
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        s[i] = soft ? exp(l[i] - top) : 1.0 / (1.0 + exp(-l[i]));
        if ((in >> i) & 1u) z += s[i];
    }
    if (soft) z = warp_sum_d(z);
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        const double dl = ((precise >> i) & 1u) || l[i] == -1.0 / 0.0 ? 0.0 : d;   // a masked expert is one for sure
        // d ln s / dl lies between 0 and 1, and so does the slope of a sigmoid's s (1 - s) in those terms
        const double e = dl == 0.0 ? 0.0 : soft ? (far ? 1.0 / 0.0 : s[i] * dl * (1.0 + dl)) : far ? 1.0 : dl * fmin(0.25, s[i] * (1.0 - s[i]) * (1.0 + dl * (1.0 + dl)));
        w[i] = s[i]; ew[i] = e;                                        // of a softmax before its division, which is the same for all
        if (soft) s[i] /= z;
        r[i] = l[i]; er[i] = dl;
        if (p.bias) {
            r[i] = (in >> i) & 1u ? s[i] + (double)p.bias[lane * VPL + i] : 0.0;
            if (r[i] != r[i]) r[i] = -1.0 / 0.0;
            er[i] = !soft ? e : all ? 0.0 : far ? 1.0 : s[i] * (dl + d) * (1.0 + dl + d);   // the sum is exact when all logits are
        }
        if (!scored) { w[i] = r[i]; ew[i] = er[i]; }
    }
    bool open = false;                                                 // a decision that exact logits could turn
    uint32_t want = 0;
    if (p.TG < p.G) {
        double worth = 0.0, low = 0.0, high = 0.0, edge = 0.0;         // lane g: group g, the ends of its interval, the least lower end among its best
        const int lanes = gs / VPL;
        const double none = -1.0 / 0.0;
        if (gs % VPL == 0 && (lanes & (lanes - 1)) == 0) {
            // a group is 2^n lanes: the two best values (with their errors) and the two best upper ends of every group at once
            double a1 = none, a2 = none, e1 = 0.0, e2 = 0.0, h1 = none, h2 = none;
            auto take = [&](double v, double e) {
                if (v > a1) { a2 = a1; e2 = e1; a1 = v; e1 = e; }
                else if (v > a2) { a2 = v; e2 = e; }
            };
            auto lift = [&](double h) {
                if (h > h1) { h2 = h1; h1 = h; }
                else if (h > h2) h2 = h;
            };
#pragma unroll
            for (int i = 0; i < VPL; i++) { take(w[i], ew[i]); lift(w[i] + ew[i]); }
            for (int k = 1; k < lanes; k <<= 1) {
                const double b1 = __shfl_xor_sync(0xffffffffu, a1, k), b2 = __shfl_xor_sync(0xffffffffu, a2, k), f1 = __shfl_xor_sync(0xffffffffu, e1, k), f2 = __shfl_xor_sync(0xffffffffu, e2, k);
                const double g1 = __shfl_xor_sync(0xffffffffu, h1, k), g2 = __shfl_xor_sync(0xffffffffu, h2, k);
                take(b1, f1); take(b2, f2);
                lift(g1); lift(g2);
            }
            const int from = min(31, lane * lanes);
            worth = __shfl_sync(0xffffffffu, two ? a1 + a2 : a1, from);
            low = __shfl_sync(0xffffffffu, two ? (a1 - e1) + (a2 - e2) : a1 - e1, from);
            edge = __shfl_sync(0xffffffffu, two ? fmin(a1 - e1, a2 - e2) : a1 - e1, from);
            high = __shfl_sync(0xffffffffu, two ? h1 + h2 : h1, from);
        } else {
            for (int g = 0; g < p.G; g++) {
                double sum = 0.0, lower = 0.0, upper = 0.0, least = 0.0;
                for (int f = 0; f < 2; f++) {                          // values, then upper ends
                    int first = -1;
                    for (int t = 0; t <= (int)two; t++) {
                        Best b{0.0, -1};
                        double e = 0.0;
#pragma unroll
                        for (int i = 0; i < VPL; i++) {
                            const double v = f ? w[i] + ew[i] : w[i];
                            const int x = lane * VPL + i;
                            if (((in >> i) & 1u) && x / gs == g && x != first && (b.i < 0 || v > b.v)) { b.v = v; b.i = x; e = ew[i]; }
                        }
                        b = warp_best(b);
                        e = __shfl_sync(0xffffffffu, e, b.i / VPL);
                        first = b.i;
                        if (f) upper += b.v;
                        else {
                            sum += b.v;
                            lower += b.v - e;
                            least = t ? fmin(least, b.v - e) : b.v - e;
                        }
                    }
                }
                if (lane == g) { worth = sum; low = lower; high = upper; edge = least; }
            }
        }
        uint32_t left = p.G == 32 ? 0xffffffffu : (1u << p.G) - 1u, groups = left;
        for (int t = 0; t < p.TG; t++) left &= ~(1u << warp_best(Best{worth, ((left >> lane) & 1u) ? lane : -1}).i);
        groups &= ~left;
        const double outside = warp_best(Best{high, ((left >> lane) & 1u) ? lane : -1}).v;
        const double inside = -warp_best(Best{-low, ((groups >> lane) & 1u) ? lane : -1}).v;
        if (inside < outside) {                                        // every group at the border: what could be among its best
            open = true;
            const uint32_t border = __ballot_sync(0xffffffffu, ((groups >> lane) & 1u) ? low < outside : ((left >> lane) & 1u) && high > inside);
            for (uint32_t rest = border; rest; rest &= rest - 1) {
                const int g = __ffs((int)rest) - 1;
                const double at = __shfl_sync(0xffffffffu, edge, g);
#pragma unroll
                for (int i = 0; i < VPL; i++)
                    if (((in >> i) & 1u) && (lane * VPL + i) / gs == g && w[i] + ew[i] >= at) want |= 1u << i;
            }
        }
#pragma unroll
        for (int i = 0; i < VPL; i++)
            if (((in >> i) & 1u) && !((groups >> ((lane * VPL + i) / gs)) & 1u)) in &= ~(1u << i);
    }
    Best mine{0.0, -1};                                                // the lane's best that is left
    auto scan = [&]() {
        mine.i = -1;
#pragma unroll
        for (int i = 0; i < VPL; i++)
            if (((in >> i) & 1u) && (mine.i < 0 || r[i] > mine.v)) { mine.v = r[i]; mine.i = lane * VPL + i; }
    };
    scan();
    int my_id = -1;
    double my_s = 0.0;
    for (int j = 0; j < p.K; j++) {
        const Best b = warp_best(mine);
        const int from = b.i / VPL;
        double sv = 0.0, low = 0.0;
        if (lane == from) {
#pragma unroll
            for (int i = 0; i < VPL; i++)
                if (lane * VPL + i == b.i) { in &= ~(1u << i); sv = s[i]; low = r[i] - er[i]; }
            scan();
        }
        sv = __shfl_sync(0xffffffffu, sv, from);
        if (lane == j) { my_id = b.i; my_s = sv; }
        if (all) continue;
        low = __shfl_sync(0xffffffffu, low, from);
        bool passes = false;                                           // one that is not taken yet could be the larger one
#pragma unroll
        for (int i = 0; i < VPL; i++)
            if (((in >> i) & 1u) && r[i] + er[i] > low) { passes = true; want |= 1u << i; }
        if (__any_sync(0xffffffffu, passes)) {
            open = true;
            if (lane == from) want |= 1u << (b.i - from * VPL);
        }
    }
    if (!open || all) {
        const double sum = p.normalize ? fmax(warp_sum_d(lane < p.K ? my_s : 0.0), 6.103515625e-5) : 1.0;
        if (lane < p.K) {
            p.ids[(size_t)row * p.K + lane] = (uint32_t)my_id;
            p.probs[(size_t)row * p.K + lane] = (float)(my_s / sum * (double)p.scale);
        }
        return 0u;
    }
    want &= ~precise;
    if (!__any_sync(0xffffffffu, want != 0)) {                         // only the softmax's sum is left to doubt
        want = ~precise;
#pragma unroll
        for (int i = 0; i < VPL; i++)
            if (lane * VPL + i >= E) want &= ~(1u << i);
        want &= (1u << VPL) - 1u;
    }
    return want;
}

// ---- 32-bit path -----------------------------------------------------------------------------------------------------
// A lane's keys carry the element's index in place of their last bits (VPL - 1 - i, so that of equal ones the lower index
// comes first): sorted once, a lane's best is its first key, and taking it is a shift. What the bits hid belongs to the
// margin below which two values are not told apart here.
template <int VPL>
__device__ __forceinline__ int expert_of(uint32_t k, int from) { return from * VPL + (int)((uint32_t)(VPL - 1) - (k & (uint32_t)(VPL - 1))); }
// the value a key stands for, to within VPL units in the last place; -inf and NaN: -inf
__device__ __forceinline__ float key_value(uint32_t k) { return k < 0x00800000u ? -INFINITY : key_rank(k); }

// What two values of a token have to differ by to be told apart in 32 bits.
struct Margin {
    float error, relative, least;            // 2 * (error of a ranking value), of its size, and near zero
    bool none;                               // the values are exact
    __device__ __forceinline__ bool near(float a, float b) const { return !none && !(a - b > error + relative * fabsf(a) + least); }   // a >= b; also two of -inf
};
// A token's row: its logits, their error, the softmax's largest one.
struct OpenRow {
    const float* logits;
    int row;
    bool bad;                                // the weights are NaN, and nothing is settled
    float error, top, inv;                   // inv: the largest score of a softmax, or 1
};
// The sum of a softmax's scores in 64 bits, where it matters: beside a bias.
template <int VPL>
__device__ __forceinline__ double softmax_sum(const SelectParams& p, const OpenRow& o, int lane) {
    if (p.score != OCO_SCORE_SOFTMAX || !p.bias) return 1.0;
    double z = 0.0;
#pragma unroll 1
    for (int i = 0; i < VPL; i++)
        if (lane * VPL + i < p.E) z += exp((double)__ldcg(o.logits + lane * VPL + i) - (double)o.top);
    return warp_sum_d(z);
}
// What a token still needs: the exact logits of the experts `want` of its lanes, and with them to
enum OpenKind {
    kDone,
    kWinners,        // put in order the winners that are too near: lane j's is not told apart from lane j - 1's where bit j of `near` is set
    kGroups,         // decide which `stay` of the groups in `near` do (`out`: the groups that go, all of those too); `group`: of the lane's expert
    kAll             // go through exact_step, as often as that wants more exact logits
};
struct Open {
    int kind, want, my_id, group, stay;
    uint32_t near, out;
};
// The lanes' exact logits where no CTA has summed them: as given, or summed by this warp.
__device__ __forceinline__ double exact_of_lanes(const SelectParams& p, const OpenRow& o, int lane, int want) {
    if (!(o.error > 0.f)) return want >= 0 ? (double)__ldcg(o.logits + want) : 0.0;
    double l = 0.0;
    for (uint32_t rest = __ballot_sync(0xffffffffu, want >= 0); rest;) {
        const int j = __ffs((int)rest) - 1;
        rest &= rest - 1;
        const int k = rest ? __ffs((int)rest) - 1 : j;
        rest &= rest - 1;
        double a, b;
        exact_logits(p, o.row, lane, __shfl_sync(0xffffffffu, want, j), __shfl_sync(0xffffffffu, want, k), a, b);
        if (lane == j) l = a;
        if (lane == k) l = b;
    }
    return l;
}
// Ranking value (score + bias, without a bias the logit) and score of a lane's expert in 64 bits. `z`: the softmax's sum.
__device__ __forceinline__ void exact_values(const SelectParams& p, const OpenRow& o, int want, double l, double z, double& r, double& v) {
    v = p.score == OCO_SCORE_SOFTMAX ? exp(l - (double)o.top) / z : 1.0 / (1.0 + exp(-l));
    r = !p.bias ? l : want >= 0 ? v + (double)p.bias[want] : 0.0;
    if (r != r) r = -1.0 / 0.0;                                        // a bias that is NaN ranks last
}
// The softmax's sum is not exact where the logits are not: what it does to the difference of two values that have scores
// va and vb in them.
__device__ __forceinline__ bool sum_matters(const SelectParams& p, const OpenRow& o, double difference, double va, double vb) {
    return o.error > 0.f && p.score == OCO_SCORE_SOFTMAX && p.bias && (o.error > kFarError || fabs(difference) <= 1.05 * (double)o.error * fabs(va - vb));
}

// Largest first (Batcher's merge exchange).
template <int N>
__device__ __forceinline__ void sort_keys(uint32_t (&k)[N]) {
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int q = p; q >= 1; q /= 2)
#pragma unroll
            for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; i++)
                    if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
                        const uint32_t a = k[i + j], b = k[i + j + q];
                        k[i + j] = max(a, b);
                        k[i + j + q] = min(a, b);
                    }
}

// Ids and weights of a token whose lane j has the j-th winner.
__device__ __forceinline__ void write_row(const SelectParams& p, const OpenRow& o, int lane, int my_id) {
    const bool soft = p.score == OCO_SCORE_SOFTMAX;
    float s = 0.f;
    if (lane < p.K) {
        const float v = __ldcg(o.logits + my_id);
        s = soft ? expf(v - o.top) * o.inv : 1.0f / (1.0f + expf(-v));
    }
    float sum = 1.0f;
    if (p.normalize) {
        sum = warp_sum_f(s);
        if (!soft || p.bias) sum = fmaxf(sum, 6.103515625e-5f);        // of a softmax's largest scores: never below top_k / experts
    }
    if (lane < p.K) {
        p.ids[(size_t)o.row * p.K + lane] = (uint32_t)my_id;
        p.probs[(size_t)o.row * p.K + lane] = o.bad ? qnan() : s / sum * p.scale;
    }
}

// A run of near winners that crosses the border takes in what is near behind it (`key`: the sorted keys that are left).
template <int VPL>
__device__ __noinline__ Open behind_border(const SelectParams& p, int lane, Margin margin, uint32_t (&key)[VPL], Open q, float mine) {
    int n = p.K + 1;
    while ((q.near >> (n - 1)) & 1u) {
        const uint32_t m = warp_max(key[0]);
        const float last = __shfl_sync(0xffffffffu, mine, n - 1), v = key_value(m);
        if (!m || !margin.near(last, v)) break;
        if (n == 32) { q.kind = kAll; break; }
        const int from = __ffs((int)__ballot_sync(0xffffffffu, key[0] == m)) - 1;
        if (lane == n) { q.my_id = expert_of<VPL>(m, from); mine = v; }
        if (lane == from) {
#pragma unroll
            for (int i = 0; i + 1 < VPL; i++) key[i] = key[i + 1];
            key[VPL - 1] = 0u;
        }
        q.near |= 1u << n++;
    }
    return q;
}

// The choice from sorted keys, without the groups in q.out; written, or left open.
template <int VPL>
__device__ __forceinline__ Open choose(const SelectParams& p, const OpenRow& o, int lane, const Margin& margin, uint32_t (&key)[VPL], Open q) {
    const int K = p.K;
    if (p.TG < p.G) {
        const int gs = p.E / p.G;
        if (gs % VPL == 0) {                                           // a lane's experts are all of one group
            if ((q.out >> min(31, lane * VPL / gs)) & 1u) {
#pragma unroll
                for (int i = 0; i < VPL; i++) key[i] = 0u;
            }
        } else {
#pragma unroll
            for (int i = 0; i < VPL; i++)
                if (key[i] && ((q.out >> (expert_of<VPL>(key[i], lane) / gs)) & 1u)) key[i] = 0u;
            sort_keys(key);
        }
    }
    // top-k: lane j keeps the j-th key and the lane it came from
    uint32_t my_key = 0;
    int my_from = 0;
    for (int j = 0; j <= K; j++) {
        const uint32_t m = warp_max(key[0]);
        const int from = __ffs((int)__ballot_sync(0xffffffffu, key[0] == m)) - 1;
        if (lane == j) { my_key = m; my_from = from; }
        if (lane == from) {
#pragma unroll
            for (int i = 0; i + 1 < VPL; i++) key[i] = key[i + 1];
            key[VPL - 1] = 0u;
        }
    }
    q.my_id = expert_of<VPL>(my_key, my_from);
    const float mine = my_key ? key_value(my_key) : 0.f, before = __shfl_up_sync(0xffffffffu, mine, 1);
    q.near = __ballot_sync(0xffffffffu, lane > 0 && lane <= K && my_key && margin.near(before, mine));
    if (q.near && !o.bad) {
        q.kind = kWinners;
        if ((q.near >> K) & 1u) {
            uint32_t left[VPL];                                        // a copy that may lie in memory
#pragma unroll
            for (int i = 0; i < VPL; i++) left[i] = key[i];
            q = behind_border<VPL>(p, lane, margin, left, q, mine);
        }
        q.want = ((q.near | (q.near >> 1)) >> lane) & 1u ? q.my_id : -1;
        return q;
    }
    q.kind = kDone;
    write_row(p, o, lane, q.my_id);
    return q;
}

// Takes an open token to its end, or to kAll; `l`: the exact logits of the lanes' experts. `key`: the sorted keys (kGroups).
template <int VPL>
__device__ __noinline__ bool settle(const SelectParams& p, OpenRow o, int lane, Margin margin, uint32_t (&key)[VPL], Open q, double l) {
    const double z = softmax_sum<VPL>(p, o, lane);
    double r, v;
    exact_values(p, o, q.want, l, z, r, v);
    if (q.kind == kGroups) {
        const bool two = p.best == 2 && p.E > p.G;
        const double part = two && !p.bias ? v : r;                    // of a group's worth
        double worth = 0.0, scores = 0.0;                              // lane g: of group g, and the scores in it
        for (uint32_t rest = q.near; rest; rest &= rest - 1) {
            const int g = __ffs((int)rest) - 1;
            const Best a = warp_best(Best{part, q.want >= 0 && q.group == g ? lane : -1});
            const Best b = warp_best(Best{part, two && q.want >= 0 && q.group == g && lane != a.i ? lane : -1});
            const double sum = two ? __shfl_sync(0xffffffffu, v, a.i) + __shfl_sync(0xffffffffu, v, b.i & 31) : __shfl_sync(0xffffffffu, v, a.i);
            if (lane == g) { worth = two ? a.v + b.v : a.v; scores = sum; }
        }
        const uint32_t border = q.near;
        uint32_t left = border;
        for (int t = 0; t < q.stay; t++) left &= ~(1u << warp_best(Best{worth, ((left >> lane) & 1u) ? lane : -1}).i);
        bool doubt = false;                                            // between one that stays and one that goes
        for (uint32_t rest = left; rest; rest &= rest - 1) {
            const int g = __ffs((int)rest) - 1;
            const double wg = __shfl_sync(0xffffffffu, worth, g), vg = __shfl_sync(0xffffffffu, scores, g);
            doubt = doubt || (((border & ~left) >> lane) & 1u && sum_matters(p, o, worth - wg, scores, vg));
        }
        if (__any_sync(0xffffffffu, doubt)) q.kind = kAll;
        else {
            q.out = (q.out & ~border) | left;
            q = choose<VPL>(p, o, lane, margin, key, q);
            if (q.kind == kWinners) exact_values(p, o, q.want, exact_of_lanes(p, o, lane, q.want), z, r, v);
        }
    }
    if (q.kind == kWinners) {
        const uint32_t members = q.near | (q.near >> 1);
        const uint32_t begins = ~q.near & ((2u << lane) - 1u);         // a run's first lane is the last one up to here that is not linked to the one before
        const int first = 31 - __clz((int)begins);
        int place = first;
        bool doubt = false;
        for (uint32_t rest = members; rest; rest &= rest - 1) {
            const int t = __ffs((int)rest) - 1;
            const int start = __shfl_sync(0xffffffffu, first, t), it = __shfl_sync(0xffffffffu, q.my_id, t);
            const double rt = __shfl_sync(0xffffffffu, r, t), vt = __shfl_sync(0xffffffffu, v, t);
            if (start != first || t == lane || !((members >> lane) & 1u)) continue;
            place += rt > r || (rt == r && it < q.my_id);
            doubt = doubt || sum_matters(p, o, r - rt, v, vt);
        }
        if (__any_sync(0xffffffffu, doubt)) q.kind = kAll;
        else {
            int id = q.my_id;
            for (uint32_t rest = members; rest; rest &= rest - 1) {
                const int t = __ffs((int)rest) - 1, to = __shfl_sync(0xffffffffu, place, t), it = __shfl_sync(0xffffffffu, q.my_id, t);
                if (lane == to) id = it;
            }
            write_row(p, o, lane, id);
        }
    }
    return q.kind == kAll;
}

// What a decision between the groups in q.near needs: their best experts, and those that could be among these.
template <int VPL>
__device__ __noinline__ Open best_of_groups(const SelectParams& p, int lane, Margin margin, const uint32_t (&key)[VPL], Open q) {
    const int gs = p.E / p.G, best = min(p.best, gs);
    q.kind = kGroups;
    int n = 0;                                                         // lanes that want an expert
    for (uint32_t rest = q.near; rest && q.kind == kGroups; rest &= rest - 1) {
        const int g = __ffs((int)rest) - 1;
        uint32_t k[VPL];
        int m = 0;                                                     // the lane's keys of the group, still in order
#pragma unroll
        for (int i = 0; i < VPL; i++) k[i] = 0u;
#pragma unroll 1
        for (int i = 0; i < VPL; i++)
            if (key[i] && expert_of<VPL>(key[i], lane) / gs == g) k[m++] = key[i];
        m = 0;
        float last = 0.f;
        for (int t = 0;; t++) {
            const uint32_t mine = m < VPL ? k[m] : 0u, a = warp_max(mine);
            if (!a || (t >= best && !margin.near(last, key_value(a)))) break;
            if (n == 32 || t == 6) { q.kind = kAll; break; }           // so many are near only where values are equal
            const int from = __ffs((int)__ballot_sync(0xffffffffu, mine == a)) - 1;
            if (lane == n) { q.want = expert_of<VPL>(a, from); q.group = g; }
            if (lane == from) m++;
            if (t < best) last = key_value(a);
            n++;
        }
    }
    return q;
}

// One token by one warp: written, or left open (`kept`: its sorted keys where the groups are). `error`: the largest error
// of its logits (0: they are exact as given).
template <int VPL>
__device__ __forceinline__ Open select_row(const SelectParams& p, int row, float error, int lane, OpenRow& o, Margin& margin, uint32_t (&kept)[VPL]) {
    constexpr uint32_t kIndex = VPL - 1;
    const int E = p.E, gs = E / p.G;
    const float* lrow = p.logits + (size_t)row * E;                     // read past L1: other CTAs of this kernel may have written them
    const bool soft = p.score == OCO_SCORE_SOFTMAX;
    // this lane's elements of E values, zero behind the last; four a load where they lie so (one a load touches every line VPL times)
    auto lane_part = [&](const float* from, float (&v)[VPL], auto load4, auto load1) {
        if (VPL >= 4 && E % 4 == 0 && ((uintptr_t)from & 15u) == 0) {
#pragma unroll
            for (int i = 0; i < VPL; i += 4) {
                float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
                if (lane * VPL + i < E) q = load4(reinterpret_cast<const float4*>(from + lane * VPL + i));
                v[i] = q.x; v[(i + 1) % VPL] = q.y; v[(i + 2) % VPL] = q.z; v[(i + 3) % VPL] = q.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < VPL; i++) v[i] = lane * VPL + i < E ? load1(from + lane * VPL + i) : 0.f;
        }
    };
    float l[VPL];
    lane_part(lrow, l, [](const float4* a) { return __ldcg(a); }, [](const float* a) { return __ldcg(a); });
    uint32_t big = 0;                                                  // largest magnitude of a logit, as bits
#pragma unroll
    for (int i = 0; i < VPL; i++) big = max(big, __float_as_uint(fabsf(l[i])));
    big = warp_max(big);
    // A logit of -inf masks its expert: its score is 0. A NaN or +inf among the logits, or nothing but -inf, makes the
    // weights NaN.
    bool any_bad = false;
    if (big >= 0x7f800000u) {
        bool bad = false, alive = false;
        uint32_t finite = 0;
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            if (lane * VPL + i >= E) continue;
            bad = bad || !(l[i] < INFINITY);
            alive = alive || l[i] > -INFINITY;
            if (!nonfinite(l[i])) finite = max(finite, __float_as_uint(fabsf(l[i])));
        }
        any_bad = __any_sync(0xffffffffu, bad) || !__any_sync(0xffffffffu, alive);
        big = warp_max(finite);
        if (any_bad) {
#pragma unroll
            for (int i = 0; i < VPL; i++)
                if (nonfinite(l[i])) l[i] = -3.4e38f;
        }
    }
    const float dl = any_bad ? 0.f : error;                            // largest error of a logit of this row (0: they are exact as given)
    const bool pairs = p.TG < p.G && p.best == 2 && gs > 1;            // groups are worth two scores
    float top = 0.f, inv = 1.f;
    if (soft) {
        float m = -3.4e38f;
#pragma unroll
        for (int i = 0; i < VPL; i++)
            if (lane * VPL + i < E) m = fmaxf(m, l[i]);
        top = key_rank(warp_max(rank_key(m)));
    }
    // What is ranked: score + bias; without a bias the logit itself, which has the same order, or, where a softmax's groups
    // are worth two scores, its distance from the largest (a score is made of the ranked value then, and its error is that
    // value's: a common offset of the logits must not enter it). ek: the largest error of a ranking value but for what
    // grows with its size, es: of a score (a softmax's relative to the largest score, which is inv).
    const bool shifted = soft && pairs && !p.bias;
    float ek = dl;
    const float es = !soft ? kSigmoidError + 0.25f * dl : dl > kFarError ? INFINITY : kScoreError + 2.1f * dl;   // a softmax's: of its logit and of the sum
    float r[VPL];
    uint32_t wide = 0;                                                 // largest magnitude of score + bias, as bits
    bool bad_bias = false;
    if (p.bias || (soft && !p.normalize)) {
        float z = 0.f;
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            if (soft) {
                r[i] = lane * VPL + i < E ? expf(l[i] - top) : 0.f;
                z += r[i];
            } else {
                r[i] = __fdividef(1.0f, 1.0f + expf(fminf(-l[i], 80.0f)));
            }
        }
        if (soft) inv = 1.0f / warp_sum_f(z);
    }
    if (p.bias) {
        float bias[VPL];
        lane_part(p.bias, bias, [](const float4* a) { return __ldg(a); }, [](const float* a) { return __ldg(a); });
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            r[i] = r[i] * inv + bias[i];
            wide = max(wide, __float_as_uint(fabsf(r[i])));
        }
        wide = warp_max(wide);
        if (wide >= 0x7f800000u) {                                     // a bias that is not finite does not widen the margins
            uint32_t finite = 0;
#pragma unroll
            for (int i = 0; i < VPL; i++)
                if (!nonfinite(r[i])) finite = max(finite, __float_as_uint(fabsf(r[i])));
            const bool nan = wide > 0x7f800000u;
            wide = warp_max(finite);
            bad_bias = nan;
        }
        ek = (soft ? inv * es : es) + kHalfUlp * __uint_as_float(wide);
    } else {
#pragma unroll
        for (int i = 0; i < VPL; i++) r[i] = shifted ? l[i] - top : l[i];
    }
    uint32_t key[VPL];
    if (any_bad || bad_bias) {                               // a NaN among the values, or a logit that ranks last
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            const uint32_t k = any_bad && l[i] == -3.4e38f ? 1u : rank_key(r[i]);
            key[i] = lane * VPL + i < E ? (max(k, 16u) & ~kIndex) | (kIndex - i) : 0u;
        }
    } else {
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            const uint32_t u = __float_as_uint(VPL == 1 ? r[i] + 0.0f : r[i]);   // where the last bits stay, the two zeros are made one
            key[i] = lane * VPL + i < E ? ((u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u)) & ~kIndex) | (kIndex - i) : 0u;
        }
    }
    sort_keys(key);
    margin = Margin{2.f * ek, 2.f * kHalfUlp * ((VPL > 1 ? 2.f * VPL : 0.f) + (shifted ? 1.f : 0.f)), VPL > 1 ? kLeast : 0.f, VPL == 1 && ek == 0.f && !shifted};
    o = OpenRow{lrow, row, any_bad, dl, top, inv};
    Open q{kDone, -1, 0, 0, 0, 0u, 0u};
    uint32_t out = 0;                                                  // groups that do not stay
    if (p.TG < p.G) {
        const bool whole = gs % VPL == 0;                              // a lane's experts are all of one group
        auto worth_of = [&](float a, float b) {                        // of ranking values; without a bias a softmax's scores relative to the largest
            if (!pairs) return a;
            if (p.bias) return a + b;
            return soft ? expf(a) + expf(b) : __fdividef(1.0f, 1.0f + expf(fminf(-a, 80.0f))) + __fdividef(1.0f, 1.0f + expf(fminf(-b, 80.0f)));
        };
        float worth = -INFINITY;                                       // lane g: group g
        const int lanes = gs / VPL;
        if (whole && (lanes & (lanes - 1)) == 0) {
            // a group is 2^n lanes: the two best of every group at once
            uint32_t m1 = key[0], m2 = VPL > 1 ? key[VPL > 1] : 0u;
            for (int d = 1; d < lanes; d <<= 1) {
                const uint32_t o1 = __shfl_xor_sync(0xffffffffu, m1, d), o2 = __shfl_xor_sync(0xffffffffu, m2, d);
                m2 = max(max(m2, o2), min(m1, o1));
                m1 = max(m1, o1);
            }
            worth = __shfl_sync(0xffffffffu, worth_of(key_value(m1), key_value(m2)), min(31, lane * lanes));
        } else {
            for (int g = 0; g < p.G; g++) {
                uint32_t m1 = 0, m2 = 0;                               // the two best of group g
#pragma unroll
                for (int i = 0; i < VPL; i++)
                    if (key[i] && expert_of<VPL>(key[i], lane) / gs == g) {
                        if (!m1) m1 = key[i];
                        else if (!m2) m2 = key[i];
                    }
                const uint32_t a = warp_max(m1);
                const int from = __ffs((int)__ballot_sync(0xffffffffu, m1 == a)) - 1;
                const uint32_t b = pairs ? warp_max(lane == from ? m2 : m1) : 0u;
                const float w = worth_of(key_value(a), key_value(b));
                if (lane == g) worth = w;
            }
        }
        const uint32_t wkey = lane < p.G ? rank_key(worth) : 0u;
        uint32_t kt = 0;
        out = p.G == 32 ? 0xffffffffu : (1u << p.G) - 1u;
        for (int t = 0; t < p.TG; t++) {
            const uint32_t mine = (out >> lane) & 1u ? wkey : 0u;
            kt = warp_max(mine);
            out &= ~(1u << (__ffs((int)__ballot_sync(0xffffffffu, mine == kt && ((out >> lane) & 1u))) - 1));
        }
        const uint32_t mine = (out >> lane) & 1u ? wkey : 0u, k2 = warp_max(mine);
        const float wa = key_rank(kt), wb = key_rank(k2);
        // error of a worth: of one value, or of two and the rounding of their sum
        const float size = !pairs ? fabsf(wa) : p.bias ? __uint_as_float(wide) : 1.f;
        const float one = (pairs && !p.bias ? es : ek) + (VPL > 1 ? 2.f * VPL * kHalfUlp * size + kLeast : 0.f) + (shifted ? 2.f : 1.f) * kHalfUlp * size;
        const float near_w = pairs ? 4.f * one : 2.f * one;
        if ((VPL > 1 || ek > 0.f || pairs) && !(wa - wb > near_w) && !any_bad) {
            // every group that could be on the other side of the border
            q.near = __ballot_sync(0xffffffffu, lane < p.G && ((out >> lane) & 1u ? !(wa - worth > near_w) : !(worth - wb > near_w)));
            q.stay = __popc(q.near & ~out);
            q.out = out;
#pragma unroll
            for (int i = 0; i < VPL; i++) kept[i] = key[i];
            return best_of_groups<VPL>(p, lane, margin, kept, q);
        }
    }
    q.out = out;
    return choose<VPL>(p, o, lane, margin, key, q);
}

// The tokens of a CTA of 256 threads, one per warp (row < 0: none). PRODUCT: logits with errors, for which the CTA sums
// what its open tokens want. Without it a warp settles its token on the spot.
template <int VPL, bool PRODUCT>
__device__ __forceinline__ void select_tokens(const SelectParams& p, int row, float error, SelectShared* sh) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    OpenRow o;
    Margin margin;
    uint32_t kept[VPL];
    Open q{kDone, -1, 0, 0, 0, 0u, 0u};
    if (row >= 0) q = select_row<VPL>(p, row, error, lane, o, margin, kept);
    if (PRODUCT ? !__syncthreads_or(q.kind != kDone) : q.kind == kDone) return;
    double l = 0.0;
    uint32_t lanes = 0;
    int at = 0;
    // the CTA sums the logits that its lanes want; each lane gets its own
    auto sum_wanted = [&](bool wants, int expert) {
        lanes = __ballot_sync(0xffffffffu, wants);
        at = __popc(lanes & ((1u << lane) - 1u));
        if (lane == 0) { sh->row[warp] = row; sh->count[warp] = __popc(lanes); }
        if (wants) sh->want[warp][at] = expert;
        __syncthreads();
        exact_wanted(p, *sh);
        double v = 0.0;
        if (wants)
            for (int w = 0; w < 8; w++) v += sh->part[w][warp][at];
        return v;
    };
    const bool some = (q.kind == kWinners || q.kind == kGroups) && q.want >= 0;
    if (PRODUCT) l = sum_wanted(some, q.want);
    else if (some) l = (double)__ldcg(o.logits + q.want);
    bool open = q.kind == kAll;
    if (q.kind == kWinners || q.kind == kGroups) open = settle<VPL>(p, o, lane, margin, kept, q, l);
    if (PRODUCT ? !__syncthreads_or(open) : !open) return;
    double all[VPL];
    uint32_t precise = 0, want = 0;
    if (open) {
#pragma unroll
        for (int i = 0; i < VPL; i++) all[i] = lane * VPL + i < p.E ? (double)__ldcg(o.logits + lane * VPL + i) : 0.0;
        if (!(o.error > 0.f)) precise = 0xffffffffu;
    }
    while (true) {
        if (open && !__any_sync(0xffffffffu, want != 0u)) {
            want = exact_step<VPL>(p, row, lane, (double)o.error, all, precise);
            open = __any_sync(0xffffffffu, want != 0u);
        }
        if (PRODUCT ? !__syncthreads_or(open) : true) return;
        const int i = __ffs((int)want) - 1;                            // one element of a lane at a time
        l = sum_wanted(open && i >= 0, lane * VPL + i);
        if (i >= 0) {
#pragma unroll
            for (int k = 0; k < VPL; k++)
                if (k == i) all[k] = l;
            want &= want - 1;
            precise |= 1u << i;
        }
    }
}

// CTAs an SM: what is bound by the latency of one row after the other gains a little from more warps than the registers of
// the usual path allow for (given logits, 32768 rows of 256 experts, 4 / 5 / 6: 44.8 / 43.9 / 43.6 us); behind the product,
// where CTAs sum exact logits, the spills weigh more (8192 rows, 3 / 4 / 5: 39.4 / 39.4 / 41.5 us).
template <int VPL, bool PRODUCT>
__global__ void __launch_bounds__(256, VPL > 8 ? 2 : PRODUCT ? 4 : 6) select_kernel(const SelectParams p) {
    __shared__ typename std::conditional<PRODUCT, SelectShared, int>::type sh;
    pdl_wait();                // the kernel before has completed and its writes are visible
    pdl_launch_dependents();
    if (__syncthreads_or(p.status && threadIdx.x == 0 && *reinterpret_cast<volatile uint32_t*>(p.status) != 0u)) return;
    const int row = blockIdx.x * 8 + (threadIdx.x >> 5);
    float error = 0.f;
    if (PRODUCT && row < p.rows)
        for (int t = 0; t < (p.E + 127) / 128; t++) error = fmaxf(error, __ldcg(p.errors + (size_t)t * p.rows + row));
    select_tokens<VPL, PRODUCT>(p, row < p.rows ? row : -1, error, reinterpret_cast<SelectShared*>(&sh));
}

// Few rows: the product and the selection in one launch. A warp per expert and four tokens makes the logits: four terms at
// a time in 32 bits, their sums in 64, which leaves a term five roundings (four, and the logit's). The CTA that comes last
// for its four tokens (counted in `arrivals`, which it leaves at zero) selects for them. No CTA waits.
template <int VPL>
__global__ void __launch_bounds__(256) route_rows_kernel(const SelectParams p, float* logits, uint32_t* arrivals) {
    __shared__ SelectShared sh;
    __shared__ int last;
    __shared__ float squares[8];
    pdl_wait();                // the kernel before has completed and its writes are visible
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, e = blockIdx.y * 8 + warp, t0 = blockIdx.x * 4;
    if (e < p.E) {
        double acc[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 4
        for (int k = lane * 4; k < p.H; k += 128) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(p.w + (size_t)e * p.H + k));
#pragma unroll
            for (int t = 0; t < 4; t++) {
                if (t0 + t >= p.rows) continue;
                const uint2 q = *reinterpret_cast<const uint2*>(p.x + (size_t)(t0 + t) * p.H + k);
                acc[t] += (double)fmaf(v.w, __uint_as_float(q.y & 0xffff0000u), fmaf(v.z, __uint_as_float(q.y << 16),
                               fmaf(v.y, __uint_as_float(q.x & 0xffff0000u), v.x * __uint_as_float(q.x << 16))));
            }
        }
        // the four sums together: half of the lanes go on with two of them, a quarter with one
        const bool upper = lane & 16, odd = lane & 8;
        double a = (upper ? acc[2] : acc[0]) + __shfl_xor_sync(0xffffffffu, upper ? acc[0] : acc[2], 16);
        double b = (upper ? acc[3] : acc[1]) + __shfl_xor_sync(0xffffffffu, upper ? acc[1] : acc[3], 16);
        a = (odd ? b : a) + __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
#pragma unroll
        for (int d = 4; d >= 1; d >>= 1) a += __shfl_xor_sync(0xffffffffu, a, d);
        const int t = lane >> 3;
        if ((lane & 7) == 0 && t0 + t < p.rows) logits[(size_t)(t0 + t) * p.E + e] = (float)a;
    }
    // the rows' squares, two warps a row (which lies in L1 by now)
    {
        const int t = t0 + (warp & 3), half = warp >> 2;
        float sq = 0.f;
        uint32_t some = 0;
        if (t < p.rows) {
#pragma unroll 4
            for (int k = (half * 32 + lane) * 8; k < p.H; k += 512) {
                const uint4 q = *reinterpret_cast<const uint4*>(p.x + (size_t)t * p.H + k);
                const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float lo = __uint_as_float(w[i] << 16), hi = __uint_as_float(w[i] & 0xffff0000u);
                    sq = fmaf(hi, hi, fmaf(lo, lo, sq));
                    some |= w[i];
                }
            }
        }
        sq = warp_sum_f(sq) + (__any_sync(0xffffffffu, (some & 0x7fff7fffu) != 0u) ? kLostSquares : 0.f);
        if (lane == 0) squares[warp] = sq;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicInc(&arrivals[blockIdx.x], gridDim.y - 1) == gridDim.y - 1;   // the last one sets the counter back to zero
        __threadfence();
    }
    __syncthreads();
    if (!last) return;
    const bool mine = warp < 4 && t0 + warp < p.rows;
    select_tokens<VPL, true>(p, mine ? t0 + warp : -1, mine ? product_error(5.1f, squares[warp] + squares[warp + 4], __ldcg(p.w_norm + 4)) : 0.f, &sh);
}

}  // namespace oco
