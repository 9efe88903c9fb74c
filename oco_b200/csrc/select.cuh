// Selection of a token's experts from its logits, with groups of experts, for one warp per token.
//
// Lane l owns the VPL consecutive experts l * VPL .. l * VPL + VPL - 1, so that the lowest lane, and within it the lowest
// element, is the lowest expert index: equal values go to the lower index without a comparison of indices.
//
// Everything is first done in 32 bits. Two ranking values that lie within each other's error (rounding of the score, of
// score + bias, and the error of the logit where it came from the router product) leave their order open; such a token
// goes through the same steps in 64 bits, where the logits that matter are summed again from x and the weights. With
// continuous logits that is a token in a few hundred, so the 64-bit path costs time only as a tail.
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

// Error of a logit that came from the router product: a sum of H products whose partial sums are of the size of the
// row's logits, taken in 32-bit accumulators (relative to the larger of the logit and the row's root mean square).
constexpr float kLogitError = 1.6e-6f;
// Relative error of a 32-bit score: two roundings and the exponential's two units in the last place, with room.
constexpr float kScoreError = 6e-7f, kHalfUlp = 6e-8f;

// ---- 64-bit path ---------------------------------------------------------------------------------------------------
struct Best { double v; int i; float e; };
// The largest value of the warp, the lowest index among equals; i = -1: no candidate.
__device__ __forceinline__ Best warp_best(Best b) {
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) {
        const double v = __shfl_xor_sync(0xffffffffu, b.v, d);
        const int i = __shfl_xor_sync(0xffffffffu, b.i, d);
        const float e = __shfl_xor_sync(0xffffffffu, b.e, d);
        if (i >= 0 && (b.i < 0 || v > b.v || (v == b.v && i < b.i))) { b.v = v; b.i = i; b.e = e; }
    }
    return b;
}

// Writes ids and weights of one token; called by a whole warp. `l`: the lane's logits, `bad`: lanes' elements whose logit
// is not finite never come here. Not inlined: it is rare and would cost the 32-bit path registers.
template <int VPL>
__device__ __noinline__ void select_exact(const SelectParams& p, int row, const float* lrow, int lane) {
    const int E = p.E, gs = p.E / p.G;
    const bool soft = p.score == OCO_SCORE_SOFTMAX, remake = p.x != nullptr;
    double l[VPL], s[VPL], r[VPL];
    float e[VPL];
    uint32_t precise = 0;                                              // bit i: element i's logit is exact
    double top = -1e300;
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        const int x = lane * VPL + i;
        l[i] = x < E ? (double)lrow[x] : 0.0;
        if (x < E) { top = fmax(top, l[i]); sq += (float)(l[i] * l[i]); }
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float rms = sqrtf(warp_sum_f(sq) / (float)E);
    if (!remake) precise = 0xffffffffu;
    else {
        // a row of zeros has exact logits, and it is what padding looks like
        uint32_t any = 0;
        const uint4* xr = reinterpret_cast<const uint4*>(p.x + (size_t)row * p.H);
        for (int k = lane; k < p.H / 8; k += 32) { const uint4 q = xr[k]; any |= (q.x | q.y | q.z | q.w) & 0x7fff7fffu; }
        if (!__any_sync(0xffffffffu, any != 0)) precise = 0xffffffffu;
    }
    while (true) {
        // scores and ranks from the present logits
        double z = 1.0;
        bool all = true;
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            const int x = lane * VPL + i;
            if (x < E && !((precise >> i) & 1u)) all = false;
            s[i] = soft ? exp(l[i] - top) : 1.0 / (1.0 + exp(-l[i]));
        }
        all = __all_sync(0xffffffffu, all);
        if (soft) {
            z = 0.0;
#pragma unroll
            for (int i = 0; i < VPL; i++)
                if (lane * VPL + i < E) z += s[i];
            z = warp_sum_d(z);
        }
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            const int x = lane * VPL + i;
            s[i] /= z;
            const float d = kLogitError * fmaxf(fabsf((float)l[i]), rms), sf = (float)s[i];
            e[i] = ((precise >> i) & 1u) ? 0.f : sf * (1.f - sf) * d * 1.01f;
            // the sum of the softmax is not exact before all logits are; it shifts ranks only against a bias
            if (soft && p.bias && !all) e[i] += sf * kLogitError * 0.25f;
            r[i] = s[i];
            if (p.bias && x < E) { r[i] = s[i] + (double)p.bias[x]; if (r[i] != r[i]) r[i] = -1.0 / 0.0; }
        }
        bool open = false;                                             // a decision that exact logits could turn
        uint32_t want = 0;
        auto group_best = [&](int g, uint32_t not_i) {                 // best element of group g, not_i: expert left out
            Best b{0.0, -1, 0.f};
#pragma unroll
            for (int i = 0; i < VPL; i++) {
                const int x = lane * VPL + i;
                if (x < E && x / gs == g && x != (int)not_i && (b.i < 0 || r[i] > b.v)) { b.v = r[i]; b.i = x; b.e = e[i]; }
            }
            return warp_best(b);
        };
        uint32_t groups = p.G == 32 ? 0xffffffffu : (1u << p.G) - 1u;
        if (p.TG < p.G) {
            double worth = 0.0, edge = 0.0;                            // lane g: group g
            float err = 0.f;
            for (int g = 0; g < p.G; g++) {
                const Best a = group_best(g, 0xffffffffu);
                Best b{0.0, -1, 0.f};
                if (p.best == 2 && gs > 1) b = group_best(g, (uint32_t)a.i);
                if (lane == g) { worth = a.v + b.v; err = a.e + b.e; edge = b.i >= 0 ? b.v : a.v; }
            }
            uint32_t left = groups;
            Best last{0.0, -1, 0.f}, next;
            for (int t = 0; t < p.TG; t++) {
                last = warp_best(Best{worth, ((left >> lane) & 1u) ? lane : -1, err});
                left &= ~(1u << last.i);
            }
            next = warp_best(Best{worth, ((left >> lane) & 1u) ? lane : -1, err});
            groups &= ~left;
            if (last.v - next.v <= (double)(last.e + next.e) && last.e + next.e > 0.f) {
                open = true;
                for (int g = 0; g < p.G; g++) {                        // every group that could lie at the border
                    const double wg = __shfl_sync(0xffffffffu, worth, g), eg = __shfl_sync(0xffffffffu, edge, g);
                    const float er = __shfl_sync(0xffffffffu, err, g);
                    if (fabs(wg - last.v) > (double)(er + 2.f * (last.e + next.e))) continue;
#pragma unroll
                    for (int i = 0; i < VPL; i++) {
                        const int x = lane * VPL + i;
                        if (x < E && x / gs == g && r[i] + e[i] >= eg - (double)er) want |= 1u << i;
                    }
                }
            }
        }
        uint32_t taken = 0;
        Best prev{0.0, -1, 0.f};
        int my_id = -1;
        double my_s = 0.0;
        for (int j = 0; j <= p.K; j++) {
            Best b{0.0, -1, 0.f};
#pragma unroll
            for (int i = 0; i < VPL; i++) {
                const int x = lane * VPL + i;
                if (x < E && ((groups >> (x / gs)) & 1u) && !((taken >> i) & 1u) && (b.i < 0 || r[i] > b.v)) { b.v = r[i]; b.i = x; b.e = e[i]; }
            }
            b = warp_best(b);
            if (b.i < 0) break;                                        // fewer experts than K + 1
            if (j > 0 && prev.v - b.v <= (double)(prev.e + b.e) && prev.e + b.e > 0.f) {
                open = true;
#pragma unroll
                for (int i = 0; i < VPL; i++) {
                    const int x = lane * VPL + i;
                    // at the border anything as near as the next one could be meant
                    if (x == prev.i || x == b.i || (j == p.K && x < E && ((groups >> (x / gs)) & 1u) && fabs(r[i] - prev.v) <= (double)(prev.e + e[i])))
                        want |= 1u << i;
                }
            }
            double sv = 0.0;
#pragma unroll
            for (int i = 0; i < VPL; i++)
                if (lane * VPL + i == b.i) { taken |= 1u << i; sv = s[i]; }
            sv = __shfl_sync(0xffffffffu, sv, b.i / VPL);
            if (lane == j && j < p.K) { my_id = b.i; my_s = sv; }
            prev = b;
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
        // sum the wanted logits again, one after the other, the warp over the row
        for (int i = 0; i < VPL; i++) {
            uint32_t lanes = __ballot_sync(0xffffffffu, ((want >> i) & 1u) && lane * VPL + i < E);
            while (lanes) {
                const int src = __ffs((int)lanes) - 1;
                lanes &= lanes - 1;
                const float4* wr = reinterpret_cast<const float4*>(p.w + (size_t)(src * VPL + i) * p.H);
                const uint2* xr = reinterpret_cast<const uint2*>(p.x + (size_t)row * p.H);
                double a0 = 0, a1 = 0, a2 = 0, a3 = 0;
#pragma unroll 4
                for (int k = lane; k < p.H / 4; k += 32) {
                    const float4 w = __ldg(wr + k);
                    const uint2 q = xr[k];
                    a0 = fma((double)w.x, (double)__uint_as_float(q.x << 16), a0);
                    a1 = fma((double)w.y, (double)__uint_as_float(q.x & 0xffff0000u), a1);
                    a2 = fma((double)w.z, (double)__uint_as_float(q.y << 16), a2);
                    a3 = fma((double)w.w, (double)__uint_as_float(q.y & 0xffff0000u), a3);
                }
                const double sum = warp_sum_d((a0 + a1) + (a2 + a3));
#pragma unroll
                for (int q = 0; q < VPL; q++)
                    if (q == i && lane == src) l[q] = sum;
            }
        }
        precise |= want;
    }
}

// ---- 32-bit path -----------------------------------------------------------------------------------------------------
template <int VPL>
__device__ __forceinline__ void select_row(const SelectParams& p, int row, int lane) {
    const int E = p.E, gs = E / p.G, K = p.K;
    const float* lrow = p.logits + (size_t)row * E;
    const bool soft = p.score == OCO_SCORE_SOFTMAX;
    float l[VPL], s[VPL];
    uint32_t key[VPL];
    if (VPL >= 4 && E % 4 == 0 && ((uintptr_t)p.logits & 15u) == 0) {
#pragma unroll
        for (int i = 0; i < VPL; i += 4) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (lane * VPL + i < E) v = *reinterpret_cast<const float4*>(lrow + lane * VPL + i);
            l[i] = v.x; l[(i + 1) % VPL] = v.y; l[(i + 2) % VPL] = v.z; l[(i + 3) % VPL] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < VPL; i++) l[i] = lane * VPL + i < E ? lrow[lane * VPL + i] : 0.f;
    }
    uint32_t bad = 0;
    float top = 0.f, sq = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        const bool in = lane * VPL + i < E;
        if (in && nonfinite(l[i])) bad |= 1u << i;
        if ((bad >> i) & 1u) l[i] = -3.4e38f;                          // ranks last; the weights become NaN below
        sq = fmaf(l[i], l[i], sq);
    }
    const bool any_bad = __any_sync(0xffffffffu, bad != 0);
    if (soft) {
        float m = -3.4e38f;
#pragma unroll
        for (int i = 0; i < VPL; i++)
            if (lane * VPL + i < E) m = fmaxf(m, l[i]);
        top = key_rank(warp_max(rank_key(m)));
        float z = 0.f;
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            const float d = l[i] - top;
            s[i] = lane * VPL + i < E ? expf(d) : 0.f;
            z += s[i];
        }
        const float inv = 1.0f / warp_sum_f(z);
#pragma unroll
        for (int i = 0; i < VPL; i++) s[i] *= inv;
    } else {
#pragma unroll
        for (int i = 0; i < VPL; i++) s[i] = 1.0f / (1.0f + expf(-l[i]));
    }
    const float rms = p.x ? sqrtf(warp_sum_f(sq) / (float)E) : 0.f;
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        const int x = lane * VPL + i;
        float r = s[i];
        if (p.bias && x < E) r += __ldg(p.bias + x);
        key[i] = x < E ? ((bad >> i) & 1u ? 1u : rank_key(r)) : 0u;
    }
    // error of a ranking value with score sv: its own roundings, and its logit's error through the score's slope.
    // softmax: exp(l - top) also carries the rounding of l - top (|ln s| bounds it up to the sum)
    auto error_of = [&](float r, float sv) {
        float er = kScoreError * sv + kHalfUlp * fabsf(r);
        if (soft) er += kHalfUlp * sv * (16.f + fabsf(__logf(fmaxf(sv, 1e-37f))));
        if (p.x) {
            const float lv = soft ? fabsf(top) + 1.f : fabsf(__logf(fmaxf(sv, 1e-37f)) - __logf(fmaxf(1.f - sv, 1e-37f)));
            er += sv * ((1.f - sv) + (soft && p.bias ? 0.25f : 0.f) + 1e-6f) * kLogitError * fmaxf(rms, lv);
        }
        return er;
    };
    bool open = false;

    uint32_t groups = 0xffffffffu;
    if (p.TG < p.G) {
        float worth = 0.f, werr = 0.f;                                 // lane g: group g
        for (int g = 0; g < p.G; g++) {
            uint32_t m1 = 0, m2 = 0;
            float s1 = 0.f, s2 = 0.f;
#pragma unroll
            for (int i = 0; i < VPL; i++) {
                const uint32_t k = (lane * VPL + i) / gs == g ? key[i] : 0u;
                if (k > m1) { m2 = m1; s2 = s1; m1 = k; s1 = s[i]; }
                else if (k > m2) { m2 = k; s2 = s[i]; }
            }
            const uint32_t a = warp_max(m1);
            const int la = __ffs((int)__ballot_sync(0xffffffffu, m1 == a)) - 1;
            float w = key_rank(a), er = error_of(w, __shfl_sync(0xffffffffu, s1, la));
            if (a <= 1u) { w = -INFINITY; er = 0.f; }                  // nothing finite in the group
            if (p.best == 2 && gs > 1) {
                if (lane == la) { m1 = m2; s1 = s2; }
                const uint32_t b = warp_max(m1);
                const int lb = __ffs((int)__ballot_sync(0xffffffffu, m1 == b)) - 1;
                const float v = b <= 1u ? -INFINITY : key_rank(b);
                er += error_of(v, __shfl_sync(0xffffffffu, s1, lb)) + kHalfUlp * fabsf(w + v);
                w += v;
            }
            if (lane == g) { worth = w; werr = er; }
        }
        const uint32_t wkey = lane < p.G ? rank_key(worth) : 0u;
        uint32_t left = p.G == 32 ? 0xffffffffu : (1u << p.G) - 1u, k = 0;
        int at = 0;
        for (int t = 0; t < p.TG; t++) {
            const uint32_t mine = (left >> lane) & 1u ? wkey : 0u;
            k = warp_max(mine);
            at = __ffs((int)__ballot_sync(0xffffffffu, mine == k && ((left >> lane) & 1u))) - 1;
            left &= ~(1u << at);
        }
        const uint32_t mine = (left >> lane) & 1u ? wkey : 0u, k2 = warp_max(mine);
        const int at2 = __ffs((int)__ballot_sync(0xffffffffu, mine == k2 && ((left >> lane) & 1u))) - 1;
        const float er = __shfl_sync(0xffffffffu, werr, at) + __shfl_sync(0xffffffffu, werr, at2);
        open = key_rank(k) - key_rank(k2) <= er;
        groups = ~left;
#pragma unroll
        for (int i = 0; i < VPL; i++)
            if (lane * VPL + i >= E || !((groups >> ((lane * VPL + i) / gs)) & 1u)) key[i] = 0u;
    }

    int my_id = 0;
    float my_s = 0.f, prev_r = 0.f, prev_e = 0.f;
    for (int j = 0; j <= K; j++) {
        uint32_t lm = 0;
#pragma unroll
        for (int i = 0; i < VPL; i++) lm = max(lm, key[i]);
        const uint32_t m = warp_max(lm);
        if (m == 0u) break;                                            // fewer experts than K + 1
        const int src = __ffs((int)__ballot_sync(0xffffffffu, lm == m)) - 1;
        int at = 0;
        float sv = 0.f;
#pragma unroll
        for (int i = VPL - 1; i >= 0; i--)
            if (key[i] == m) { at = i; sv = s[i]; }
        if (lane == src) {
#pragma unroll
            for (int i = 0; i < VPL; i++)
                if (i == at) key[i] = 0u;
        }
        at = __shfl_sync(0xffffffffu, at, src);
        sv = __shfl_sync(0xffffffffu, sv, src);
        const float r = key_rank(m), er = error_of(r, sv);
        if (j > 0 && prev_r - r <= prev_e + er) open = true;
        prev_r = r; prev_e = er;
        if (lane == j && j < K) { my_id = src * VPL + at; my_s = sv; }
    }
    if (open && !any_bad) {
        select_exact<VPL>(p, row, lrow, lane);
        return;
    }
    float sum = 1.0f;
    if (p.normalize) sum = fmaxf(warp_sum_f(lane < K ? my_s : 0.f), 6.103515625e-5f);
    if (lane < K) {
        p.ids[(size_t)row * K + lane] = (uint32_t)my_id;
        p.probs[(size_t)row * K + lane] = any_bad ? qnan() : my_s / sum * p.scale;
    }
}

// A warp per token, eight tokens per CTA.
template <int VPL>
__global__ void __launch_bounds__(256) select_kernel(const SelectParams p) {
    pdl_launch_dependents();   // the next kernel of the step may be set up beside this one
    pdl_wait();                // the kernel before has completed and its writes are visible
    if (p.status && *reinterpret_cast<volatile uint32_t*>(p.status) != 0u) return;
    const int row = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row < p.rows) select_row<VPL>(p, row, threadIdx.x & 31);
}

}  // namespace oco
