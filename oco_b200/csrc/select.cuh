// Selection of a token's experts from its logits, with groups of experts, for one warp per token.
//
// Lane l owns the VPL consecutive experts l * VPL .. l * VPL + VPL - 1, so that the lowest lane, and within it the lowest
// element, is the lowest expert index: equal values go to the lower index without a comparison of indices.
//
// Everything is first done in 32 bits. Two ranking values that lie within each other's error (rounding of the score, of
// score + bias, and the error of the logit where it came from the router product) leave their order open; such a token
// is settled in 64 bits, where the logits that matter are summed again from x and the weights by the whole CTA (one warp
// alone took 10 to 20 us for it). With continuous logits that is a token in a few hundred.
#pragma once
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

// Error of a logit that came from the router product, relative to the largest logit of its row: a sum of exact products
// whose partial sums are of the size of the row's logits, in 32-bit accumulators.
constexpr float kLogitError = 1.5e-6f;
// A sigmoid in 32 bits: s (1 - s) 2^-22 from the exponential's two units in the last place, the sum's rounding and the
// quotient's two units: below 4e-7.
// A softmax score relative to the largest one: the same and the rounding of l - top (x e^-x < 0.37), the sum and its
// reciprocal. kHalfUlp: the rounding of score + bias.
// kLeast: 2^-126, below which the last bits of a value (an index stands there in a sorted key) weigh more than its size tells.
constexpr float kSigmoidError = 4e-7f, kScoreError = 6e-7f, kHalfUlp = 6e-8f, kLeast = 1.1754944e-38f;

// ---- exact logits, summed by a whole CTA ------------------------------------------------------------------------------
struct SelectShared {
    int rows[8];                 // rows of the CTA's warps that need exact logits, -1: none
    int row, a, b, work;         // what is asked for: the logits of experts a and b of a row; work 0: nothing more
    double part[2][8];
};
__device__ __forceinline__ void dots_share(const SelectParams& p, SelectShared* sh) {
    const float4* wa = reinterpret_cast<const float4*>(p.w + (size_t)sh->a * p.H);
    const float4* wb = reinterpret_cast<const float4*>(p.w + (size_t)sh->b * p.H);
    const uint2* xr = reinterpret_cast<const uint2*>(p.x + (size_t)sh->row * p.H);
    double a0 = 0, a1 = 0, b0 = 0, b1 = 0;
#pragma unroll 2
    for (int k = threadIdx.x; k < p.H / 4; k += 256) {
        const float4 u = __ldg(wa + k), v = __ldg(wb + k);
        const uint2 q = xr[k];
        const double x0 = (double)__uint_as_float(q.x << 16), x1 = (double)__uint_as_float(q.x & 0xffff0000u);
        const double x2 = (double)__uint_as_float(q.y << 16), x3 = (double)__uint_as_float(q.y & 0xffff0000u);
        a0 = fma((double)u.x, x0, a0); a1 = fma((double)u.y, x1, a1); a0 = fma((double)u.z, x2, a0); a1 = fma((double)u.w, x3, a1);
        b0 = fma((double)v.x, x0, b0); b1 = fma((double)v.y, x1, b1); b0 = fma((double)v.z, x2, b0); b1 = fma((double)v.w, x3, b1);
    }
    const double da = warp_sum_d(a0 + a1), db = warp_sum_d(b0 + b1);
    if ((threadIdx.x & 31) == 0) { sh->part[0][threadIdx.x >> 5] = da; sh->part[1][threadIdx.x >> 5] = db; }
}
// Warp 0 asks, the other warps wait in dots_serve.
__device__ __noinline__ void dots_ask(const SelectParams& p, SelectShared* sh, int row, int a, int b, double& da, double& db) {
    if (threadIdx.x == 0) { sh->row = row; sh->a = a; sh->b = b; sh->work = 1; }
    __syncthreads();
    dots_share(p, sh);
    __syncthreads();
    da = db = 0.0;
    for (int w = 0; w < 8; w++) { da += sh->part[0][w]; db += sh->part[1][w]; }
}
__device__ __noinline__ void dots_serve(const SelectParams& p, SelectShared* sh) {
    while (true) {
        __syncthreads();
        if (!sh->work) return;
        dots_share(p, sh);
        __syncthreads();
    }
}
__device__ __forceinline__ void dots_end(SelectShared* sh) {
    if (threadIdx.x == 0) sh->work = 0;
    __syncthreads();
}

// ---- 64-bit path ---------------------------------------------------------------------------------------------------
struct Best { double v; int i; };
// The largest value of the warp, the lowest index among equals; i = -1: no candidate.
__device__ __forceinline__ Best warp_best(Best b) {
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) {
        const double v = __shfl_xor_sync(0xffffffffu, b.v, d);
        const int i = __shfl_xor_sync(0xffffffffu, b.i, d);
        if (i >= 0 && (b.i < 0 || v > b.v || (v == b.v && i < b.i))) { b.v = v; b.i = i; }
    }
    return b;
}

// Writes ids and weights of one token; called by a whole warp. `d`: the largest error of a logit (0 without `sh`). Every
// value is held with its error, and what is decided between two values is settled when their intervals do not overlap;
// the logits of those that do are summed again. Ranked is score + bias, without a bias the logit itself: scores that
// have run into 0 or 1 keep the order of their logits. Not inlined: it is rare and would cost the 32-bit path registers.
template <int VPL>
__device__ __noinline__ void select_exact(const SelectParams& p, int row, const float* lrow, int lane, double d, SelectShared* sh) {
    const int E = p.E, gs = p.E / p.G;
    const bool soft = p.score == OCO_SCORE_SOFTMAX, remake = sh != nullptr;
    const bool scored = !p.bias && p.best == 2 && gs > 1;              // groups are worth scores, experts are ranked by logits
    double l[VPL], s[VPL], r[VPL], er[VPL], w[VPL], ew[VPL];           // logit, score, rank and part of a group's worth with their errors
    uint32_t precise = remake ? 0u : 0xffffffffu;                      // bit i: element i's logit is exact
    double top = -1.0 / 0.0;
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        const int x = lane * VPL + i;
        l[i] = x < E ? (double)__ldcg(lrow + x) : 0.0;
        if (x < E) top = fmax(top, l[i]);
    }
#pragma unroll
    for (int k = 16; k >= 1; k >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, k));
    while (true) {
        // scores, ranks and errors from the present logits
        double z = 0.0;
        bool all = true;
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            const int x = lane * VPL + i;
            if (x < E && !((precise >> i) & 1u)) all = false;
            s[i] = soft ? exp(l[i] - top) : 1.0 / (1.0 + exp(-l[i]));
            if (x < E) z += s[i];
        }
        all = __all_sync(0xffffffffu, all);
        z = soft ? warp_sum_d(z) : 1.0;
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            const int x = lane * VPL + i;
            const double dl = (precise >> i) & 1u || l[i] == -1.0 / 0.0 ? 0.0 : d;   // a masked expert is one for sure
            // d ln s / dl lies between 0 and 1, and so does the slope of a sigmoid's s (1 - s) in those terms; scores lie in 0 .. 1
            const double e = soft ? (d > 1.0 ? (dl > 0.0 ? 1.0 / 0.0 : 0.0) : s[i] * expm1(dl))
                                  : (d > 1.0 ? (dl > 0.0 ? 1.0 : 0.0) : dl * fmin(0.25, s[i] * (1.0 - s[i]) * exp(dl)));
            w[i] = s[i]; ew[i] = e;                                    // of a softmax before its division, which is the same for all
            s[i] /= z;
            r[i] = l[i]; er[i] = dl;
            if (p.bias) {
                r[i] = x < E ? s[i] + (double)p.bias[x] : 0.0;
                if (r[i] != r[i]) r[i] = -1.0 / 0.0;
                er[i] = !soft ? e : all ? 0.0 : d > 1.0 ? 1.0 : s[i] * expm1(dl + d);   // the sum is exact when all logits are
            }
            if (!scored) { w[i] = r[i]; ew[i] = er[i]; }
        }
        bool open = false;                                             // a decision that exact logits could turn
        uint32_t want = 0;
        // sum of the p.best largest w + f * ew of group g; `last`: the smaller one of them
        auto worth_of = [&](int g, double f, double& last) {
            int first = -1;
            double sum = 0.0;
            for (int t = 0; t < min(p.best, gs); t++) {
                Best b{0.0, -1};
#pragma unroll
                for (int i = 0; i < VPL; i++) {
                    const int x = lane * VPL + i;
                    const double v = f == 0.0 ? w[i] : w[i] + f * ew[i];
                    if (x < E && x / gs == g && x != first && (b.i < 0 || v > b.v)) { b.v = v; b.i = x; }
                }
                b = warp_best(b);
                first = b.i;
                last = b.v;
                sum += b.v;
            }
            return sum;
        };
        uint32_t groups = p.G == 32 ? 0xffffffffu : (1u << p.G) - 1u;
        if (p.TG < p.G) {
            double worth = 0.0, low = 0.0, high = 0.0, edge = 0.0;     // lane g: group g
            for (int g = 0; g < p.G; g++) {
                double last, e;
                const double a = worth_of(g, 0.0, last), b = worth_of(g, -1.0, e), c = worth_of(g, 1.0, last);
                if (lane == g) { worth = a; low = b; high = c; edge = e; }
            }
            uint32_t left = groups;
            for (int t = 0; t < p.TG; t++) left &= ~(1u << warp_best(Best{worth, ((left >> lane) & 1u) ? lane : -1}).i);
            groups &= ~left;
            const double out = warp_best(Best{high, ((left >> lane) & 1u) ? lane : -1}).v;
            const double in = -warp_best(Best{-low, ((groups >> lane) & 1u) ? lane : -1}).v;
            if (in < out) {
                open = true;
                for (int g = 0; g < p.G; g++) {                        // every group at the border: what could be among its best
                    const double lg = __shfl_sync(0xffffffffu, low, g), hg = __shfl_sync(0xffffffffu, high, g), eg = __shfl_sync(0xffffffffu, edge, g);
                    if ((groups >> g) & 1u ? !(lg < out) : !(hg > in)) continue;
#pragma unroll
                    for (int i = 0; i < VPL; i++) {
                        const int x = lane * VPL + i;
                        if (x < E && x / gs == g && w[i] + ew[i] >= eg) want |= 1u << i;
                    }
                }
            }
        }
        uint32_t taken = 0;
        int my_id = -1;
        double my_s = 0.0;
        for (int j = 0; j < p.K; j++) {
            Best b{0.0, -1};
#pragma unroll
            for (int i = 0; i < VPL; i++) {
                const int x = lane * VPL + i;
                if (x < E && ((groups >> (x / gs)) & 1u) && !((taken >> i) & 1u) && (b.i < 0 || r[i] > b.v)) { b.v = r[i]; b.i = x; }
            }
            b = warp_best(b);
            double sv = 0.0, low = 0.0;
#pragma unroll
            for (int i = 0; i < VPL; i++)
                if (lane * VPL + i == b.i) { taken |= 1u << i; sv = s[i]; low = r[i] - er[i]; }
            sv = __shfl_sync(0xffffffffu, sv, b.i / VPL);
            low = __shfl_sync(0xffffffffu, low, b.i / VPL);
            if (lane == j) { my_id = b.i; my_s = sv; }
            bool passes = false;                                       // one that is not taken yet could be the larger one
#pragma unroll
            for (int i = 0; i < VPL; i++) {
                const int x = lane * VPL + i;
                if (x < E && ((groups >> (x / gs)) & 1u) && !((taken >> i) & 1u) && r[i] + er[i] > low) { passes = true; want |= 1u << i; }
            }
            if (__any_sync(0xffffffffu, passes)) {
                open = true;
#pragma unroll
                for (int i = 0; i < VPL; i++)
                    if (lane * VPL + i == b.i) want |= 1u << i;
            }
        }
        want &= ~precise;
        if (open && !all && !__any_sync(0xffffffffu, want != 0)) want = ~precise;   // only the softmax's sum is left to doubt
        if (!open || !remake || all) {
            const double sum = p.normalize ? fmax(warp_sum_d(lane < p.K ? my_s : 0.0), 6.103515625e-5) : 1.0;
            if (lane < p.K) {
                p.ids[(size_t)row * p.K + lane] = (uint32_t)my_id;
                p.probs[(size_t)row * p.K + lane] = (float)(my_s / sum * (double)p.scale);
            }
            return;
        }
        // sum the wanted logits again, two at a time
        int first = -1;
        auto keep = [&](int x, double v) {
#pragma unroll
            for (int q = 0; q < VPL; q++)
                if (lane * VPL + q == x) l[q] = v;
        };
        for (int i = 0; i < VPL; i++) {
            uint32_t lanes = __ballot_sync(0xffffffffu, ((want >> i) & 1u) && lane * VPL + i < E);
            while (lanes) {
                const int x = (__ffs((int)lanes) - 1) * VPL + i;
                lanes &= lanes - 1;
                if (first < 0) { first = x; continue; }
                double da, db;
                dots_ask(p, sh, row, first, x, da, db);
                keep(first, da);
                keep(x, db);
                first = -1;
            }
        }
        if (first >= 0) {
            double da, db;
            dots_ask(p, sh, row, first, first, da, db);
            keep(first, da);
        }
        precise |= want;
    }
}

// ---- 32-bit path -----------------------------------------------------------------------------------------------------
// The ranking values r (score + bias, without a bias the logit) and scores s of two experts in 64 bits, made by a whole
// warp. `z`: the softmax's sum.
__device__ __noinline__ void exact_pair(const SelectParams& p, SelectShared* sh, int row, const float* lrow, int lane, int a, int b, double top, double z, double (&r)[2], double (&s)[2]) {
    double la = (double)__ldcg(lrow + a), lb = (double)__ldcg(lrow + b);
    if (sh) dots_ask(p, sh, row, a, b, la, lb);
    // lane 0 takes a, lane 1 takes b
    const double l = lane == 0 ? la : lb;
    const double v = p.score == OCO_SCORE_SOFTMAX ? exp(l - top) / z : 1.0 / (1.0 + exp(-l));
    const double w = p.bias ? v + (double)p.bias[lane == 0 ? a : b] : l;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        r[i] = __shfl_sync(0xffffffffu, w, i);
        s[i] = __shfl_sync(0xffffffffu, v, i);
    }
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

// A lane's keys carry the element's index in place of their last bits (VPL - 1 - i, so that of equal ones the lower index
// comes first): sorted once, a lane's best is its first key, and taking it is a shift. What the bits hid belongs to the
// margin below which two values are not told apart here.
//
// Returns 0, or, before anything is written, what an open decision needs (only where !EXACT): 1 the exact values of the
// logits as they are, 2 exact logits too. EXACT settles it: with `sh`, warp 0 while the others serve, else any warp.
template <int VPL, bool EXACT>
__device__ __forceinline__ int select_row(const SelectParams& p, int row, int lane, SelectShared* sh) {
    constexpr uint32_t kIndex = VPL - 1;
    const int E = p.E, gs = E / p.G, K = p.K;
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
    // largest error of a logit of this row (0: they are exact as given)
    const float dl = p.x && !any_bad ? kLogitError * __uint_as_float(big) : 0.f;   // rows of zeros have exact ones
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
    const float es = soft ? kScoreError + dl : kSigmoidError + 0.25f * dl;
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
    // the value a key stands for, to within VPL units in the last place; -inf and NaN: -inf
    auto value = [&](uint32_t k) { return k < 0x00800000u ? -INFINITY : key_rank(k); };
    auto margin = [&](float v) { return 2.f * ek + 2.f * kHalfUlp * fabsf(v) * ((VPL > 1 ? 2.f * VPL : 0.f) + (shifted ? 1.f : 0.f)) + (VPL > 1 ? kLeast : 0.f); };
    // two values, the first not below the second, that are not told apart (also two of -inf)
    auto too_near = [&](float a, float b) { return (VPL > 1 || ek > 0.f || shifted) && !(a - b > margin(a)); };
    auto expert_of = [&](uint32_t k, int from) { return from * VPL + (int)(kIndex - (k & kIndex)); };
    double z64 = 0.0;                                                  // the softmax's sum in 64 bits, made when it is needed
    auto sum64 = [&]() {
        if (!soft || z64 != 0.0) return;
        double z = 0.0;
#pragma unroll
        for (int i = 0; i < VPL; i++)
            if (lane * VPL + i < E) z += exp((double)__ldcg(lrow + lane * VPL + i) - (double)top);
        z64 = warp_sum_d(z);
    };

    bool open = false;                                                 // left to select_exact
    if (p.TG < p.G) {
        const bool whole = gs % VPL == 0;                              // a lane's experts are all of one group
        // the three best of group g: values, and the experts of the first two
        auto best_of = [&](int g, float (&v)[3], int (&id)[2]) {
            uint32_t m[3] = {0, 0, 0};
#pragma unroll
            for (int i = 0; i < VPL; i++)
                if (key[i] && expert_of(key[i], lane) / gs == g) {
                    if (!m[0]) m[0] = key[i];
                    else if (!m[1]) m[1] = key[i];
                    else if (!m[2]) m[2] = key[i];
                }
#pragma unroll
            for (int t = 0; t < 3; t++) {
                const uint32_t a = warp_max(m[0]);
                const int from = __ffs((int)__ballot_sync(0xffffffffu, m[0] == a)) - 1;
                v[t] = a ? value(a) : -INFINITY;
                if (t < 2) id[t] = a ? expert_of(a, from) : g * gs;
                if (lane == from) { m[0] = m[1]; m[1] = m[2]; m[2] = 0; }
            }
        };
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
            worth = __shfl_sync(0xffffffffu, worth_of(value(m1), value(m2)), min(31, lane * lanes));
        } else {
            for (int g = 0; g < p.G; g++) {
                float v[3];
                int id[2];
                best_of(g, v, id);
                const float w = worth_of(v[0], v[1]);
                if (lane == g) worth = w;
            }
        }
        const uint32_t wkey = lane < p.G ? rank_key(worth) : 0u;
        uint32_t left = p.G == 32 ? 0xffffffffu : (1u << p.G) - 1u, kprev = 0, kt = 0;
        int at = 0;
        for (int t = 0; t < p.TG; t++) {
            const uint32_t mine = (left >> lane) & 1u ? wkey : 0u;
            kprev = kt;
            kt = warp_max(mine);
            at = __ffs((int)__ballot_sync(0xffffffffu, mine == kt && ((left >> lane) & 1u))) - 1;
            left &= ~(1u << at);
        }
        const uint32_t mine = (left >> lane) & 1u ? wkey : 0u, k2 = warp_max(mine);
        const int at2 = __ffs((int)__ballot_sync(0xffffffffu, mine == k2 && ((left >> lane) & 1u))) - 1;
        const float wa = key_rank(kt), wb = key_rank(k2);
        // error of a worth: of one value, or of two and the rounding of their sum
        const float size = !pairs ? fabsf(wa) : p.bias ? __uint_as_float(wide) : 1.f;
        const float one = (pairs && !p.bias ? es : ek) + (VPL > 1 ? 2.f * VPL * kHalfUlp * size + kLeast : 0.f) + (shifted ? 2.f : 1.f) * kHalfUlp * size;
        const float near_w = pairs ? 4.f * one : 2.f * one;
        if ((VPL > 1 || ek > 0.f || pairs) && !(wa - wb > near_w) && !any_bad) {
            // the border lies between two groups: their exact worths decide, unless a third one is as near or what a group
            // is worth is not clear
            if constexpr (!EXACT) return dl > 0.f ? 2 : 1;
            const uint32_t k3 = warp_max((left >> lane) & 1u && lane != at2 ? wkey : 0u);
            open = (p.TG > 1 && !(key_rank(kprev) - wb > near_w)) || (k3 != 0u && !(wa - key_rank(k3) > near_w));
            if (!open) {
                float a[3], b[3];
                int ia[2], ib[2];
                best_of(at, a, ia);
                best_of(at2, b, ib);
                const int t = pairs ? 1 : 0;
                open = (gs > t + 1 && (too_near(a[t], a[t + 1]) || too_near(b[t], b[t + 1])));
                if (!open) {
                    sum64();
                    double r1[2], v1[2], r2[2] = {0.0, 0.0}, v2[2] = {0.0, 0.0};
                    exact_pair(p, sh, row, lrow, lane, ia[0], ib[0], (double)top, z64, r1, v1);
                    if (pairs) exact_pair(p, sh, row, lrow, lane, ia[1], ib[1], (double)top, z64, r2, v2);
                    const bool scored = pairs && !p.bias;
                    const double da = scored ? v1[0] + v2[0] : r1[0] + r2[0], db = scored ? v1[1] + v2[1] : r1[1] + r2[1];
                    // the softmax's sum is not exact where the logits are not: it shifts the scores' difference
                    if (sh && soft && p.bias && fabs(da - db) <= (double)dl * fabs((v1[0] + v2[0]) - (v1[1] + v2[1]))) open = true;
                    else if (db > da || (db == da && at2 < at)) left = (left | (1u << at)) & ~(1u << at2);
                }
            }
        }
        if (whole) {
            if ((left >> min(31, lane * VPL / gs)) & 1u) {
#pragma unroll
                for (int i = 0; i < VPL; i++) key[i] = 0u;
            }
        } else {
#pragma unroll
            for (int i = 0; i < VPL; i++)
                if (key[i] && ((left >> (expert_of(key[i], lane) / gs)) & 1u)) key[i] = 0u;
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
    int my_id = expert_of(my_key, my_from);
    const float mine = my_key ? value(my_key) : 0.f, before = __shfl_up_sync(0xffffffffu, mine, 1);
    uint32_t near = __ballot_sync(0xffffffffu, lane > 0 && lane <= K && my_key && too_near(before, mine));   // bit j: not told apart from j - 1
    if (near && !any_bad && !open) {
        if constexpr (!EXACT) return dl > 0.f ? 2 : 1;
        // neighbours that are too near change places if their exact values say so; three in a row go to select_exact
        open = (near & (near << 1)) != 0u;
        if ((near >> K) & 1u) {
            const uint32_t m = warp_max(key[0]);                       // the next one behind the border
            open = open || (m != 0u && too_near(__shfl_sync(0xffffffffu, mine, K), value(m)));
        }
        if (!open) {
            sum64();
            while (near) {
                const int j = __ffs((int)near) - 1;
                near &= near - 1;
                const int a = __shfl_sync(0xffffffffu, my_id, j - 1), b = __shfl_sync(0xffffffffu, my_id, j);
                double rr[2], v[2];
                exact_pair(p, sh, row, lrow, lane, a, b, (double)top, z64, rr, v);
                if (sh && soft && p.bias && fabs(rr[0] - rr[1]) <= (double)dl * fabs(v[0] - v[1])) open = true;
                if (rr[1] > rr[0] || (rr[1] == rr[0] && b < a)) {
                    if (lane == j - 1) my_id = b;
                    if (lane == j) my_id = a;
                }
            }
        }
    }
    if (EXACT && open) {
        select_exact<VPL>(p, row, lrow, lane, (double)dl, sh);
        return 0;
    }
    float s = 0.f;
    if (lane < K) {
        const float v = __ldcg(lrow + my_id);
        s = soft ? expf(v - top) * inv : 1.0f / (1.0f + expf(-v));
    }
    float sum = 1.0f;
    if (p.normalize) {
        sum = warp_sum_f(s);
        if (!soft || p.bias) sum = fmaxf(sum, 6.103515625e-5f);        // of a softmax's largest scores: never below top_k / experts
    }
    if (lane < K) {
        p.ids[(size_t)row * K + lane] = (uint32_t)my_id;
        p.probs[(size_t)row * K + lane] = any_bad ? qnan() : s / sum * p.scale;
    }
    return 0;
}

template <int VPL>
__device__ __noinline__ void settle_row(const SelectParams& p, int row, int lane, SelectShared* sh) { select_row<VPL, true>(p, row, lane, sh); }

// The tokens of a CTA of 256 threads, one per warp (row < 0: none). PRODUCT: the logits come from rows and weights.
template <int VPL, bool PRODUCT>
__device__ __forceinline__ void select_tokens(const SelectParams& p, int row, SelectShared& sh) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int left = row >= 0 ? select_row<VPL, false>(p, row, lane, nullptr) : 0;
    if (left == 1) settle_row<VPL>(p, row, lane, nullptr);
    if (!PRODUCT || !__syncthreads_or(left == 2)) return;
    if (lane == 0) sh.rows[warp] = left == 2 ? row : -1;
    __syncthreads();
    if (warp == 0) {
        for (int w = 0; w < 8; w++)
            if (sh.rows[w] >= 0) settle_row<VPL>(p, sh.rows[w], lane, &sh);
        dots_end(&sh);
    } else {
        dots_serve(p, &sh);
    }
}

// CTAs an SM: what is bound by the latency of one row after the other gains from more warps than the registers of the
// usual path allow for (given logits, 32768 rows of 256 experts, 4 / 5 / 6: 49.8 / 47.7 / 46.5 us); behind the product,
// where CTAs wait for exact logits, the spills weigh more (8192 rows with their product 85.2 / 85.9 / 87.8 us).
template <int VPL, bool PRODUCT>
__global__ void __launch_bounds__(256, VPL > 8 ? 2 : PRODUCT ? 4 : 6) select_kernel(const SelectParams p) {
    __shared__ SelectShared sh;
    pdl_wait();                // the kernel before has completed and its writes are visible
    pdl_launch_dependents();
    if (__syncthreads_or(p.status && threadIdx.x == 0 && *reinterpret_cast<volatile uint32_t*>(p.status) != 0u)) return;
    const int row = blockIdx.x * 8 + (threadIdx.x >> 5);
    select_tokens<VPL, PRODUCT>(p, row < p.rows ? row : -1, sh);
}

// Few rows: the product and the selection in one launch. A warp per expert and four tokens makes the logits (f32); the CTA
// that comes last for its four tokens (counted in `arrivals`, which it leaves at zero) selects for them. No CTA waits.
template <int VPL>
__global__ void __launch_bounds__(256) route_rows_kernel(const SelectParams p, float* logits, uint32_t* arrivals) {
    __shared__ SelectShared sh;
    __shared__ int last;
    pdl_wait();                // the kernel before has completed and its writes are visible
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, e = blockIdx.y * 8 + warp, t0 = blockIdx.x * 4;
    if (e < p.E) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int k = lane * 4; k < p.H; k += 128) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(p.w + (size_t)e * p.H + k));
#pragma unroll
            for (int t = 0; t < 4; t++) {
                if (t0 + t >= p.rows) continue;
                const uint2 q = *reinterpret_cast<const uint2*>(p.x + (size_t)(t0 + t) * p.H + k);
                acc[t] = fmaf(v.x, __uint_as_float(q.x << 16), acc[t]);
                acc[t] = fmaf(v.y, __uint_as_float(q.x & 0xffff0000u), acc[t]);
                acc[t] = fmaf(v.z, __uint_as_float(q.y << 16), acc[t]);
                acc[t] = fmaf(v.w, __uint_as_float(q.y & 0xffff0000u), acc[t]);
            }
        }
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const float s = warp_sum_f(acc[t]);
            if (lane == 0 && t0 + t < p.rows) logits[(size_t)(t0 + t) * p.E + e] = s;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicInc(&arrivals[blockIdx.x], gridDim.y - 1) == gridDim.y - 1;   // the last one sets the counter back to zero
        __threadfence();
    }
    __syncthreads();
    if (!last) return;
    select_tokens<VPL, true>(p, warp < 4 && t0 + warp < p.rows ? t0 + warp : -1, sh);
}

}  // namespace oco
