// The step between two blocks of a layer, in one pass over the rows: the finished block's output is normalised
// (post-norm, optional), gated and scaled onto the residual rows, and the result is normalised for the next block:
//
//     b  = post(block)                          RMS:   v * rsqrt(mean(v^2) + eps) * (offset + w)
//     h  = residual_scale * hidden              layer: (v - mean(v)) * rsqrt(var(v) + eps) * (offset + w) + bias
//        + block_scale * act(gate) * b
//     x  = pre(h)
//
// Bound: memory. Rows are read once and written once (hidden, block and a per-element gate in; hidden and x out); a
// row lives in the registers of the threads that share it, so the statistics cost no second read. They are sums in
// f32; the variance of the layer form is the mean square of the centred values (two sums over registers), not a
// difference of large sums. x is made from the f32 value of h, not from its rounded copy: one rounding per output.
#include "host.cuh"

using namespace oco;

namespace {

constexpr int kMaxWidth = 32768;

struct NormParams {
    const void* hidden;
    const uint16_t* block;
    const float *post_w, *post_b, *pre_w, *pre_b;
    const void* gate;
    void* hidden_out;
    uint16_t* norm_out;
    long long hidden_stride, block_stride, gate_stride, hidden_out_stride, norm_out_stride;
    int n, rows, gate_type, gate_rows, gate_act;
    float eps, offset, residual_scale, block_scale;
};

// Eight elements are four pairs of f32: the packed operations take half the instructions, and instructions are what
// bounds a kernel with two norms and a gate (measured with scalar ones: issue slots 67 % busy, memory 59 %).
struct Oct { uint64_t v[4]; };
__device__ __forceinline__ Oct unpack8(const uint4& q) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    Oct r;
#pragma unroll
    for (int j = 0; j < 4; j++) r.v[j] = f32x2_bits(w[j] << 16, w[j] & 0xffff0000u);
    return r;
}
__device__ __forceinline__ Oct pairs8(const uint4& a, const uint4& b) {
    return Oct{{f32x2_bits(a.x, a.y), f32x2_bits(a.z, a.w), f32x2_bits(b.x, b.y), f32x2_bits(b.z, b.w)}};
}
__device__ __forceinline__ uint4 pack8(const Oct& r) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float lo, hi;
        f32x2_split(r.v[j], lo, hi);
        const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
        w[j] = *reinterpret_cast<const uint32_t*>(&p);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ Oct load8(const float* p) {
    return pairs8(__ldg(reinterpret_cast<const uint4*>(p)), __ldg(reinterpret_cast<const uint4*>(p) + 1));
}
// The same of an array that a kernel before in the stream may have written.
__device__ __forceinline__ Oct fetch8(const float* p) { return pairs8(*reinterpret_cast<const uint4*>(p), *(reinterpret_cast<const uint4*>(p) + 1)); }
// To four or five units in the last place: the quotient's two are below the clamp's limit, where 1 + e^87 is still in its
// range (8192 rows of 4096: 72 us, with the hardware's exponential, which is off by a unit for each unit of x, 68, with a
// rounded quotient 78). A NaN stays one.
__device__ __forceinline__ float gate_sigmoid(float x) { return __fdividef(1.0f, 1.0f + expf(x < -87.0f ? 87.0f : -x)); }
__device__ __forceinline__ uint64_t both(float v) { return f32x2(v, v); }
__device__ __forceinline__ float sum2(uint64_t v) {
    float lo, hi;
    f32x2_split(v, lo, hi);
    return lo + hi;
}

// Sum over the THREADS threads that share a row; every one of them gets it. `slot`: shared memory, a fresh one per call.
template <int THREADS>
__device__ __forceinline__ float row_sum(float s, float* slot) {
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (THREADS == 32) return s;
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = s;
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < THREADS / 32; i++) t += slot[i];
    return t;
}

// Normalises the row held in v (elements at or past n are zero and stay out of the sums). LAYER: centred first.
template <int THREADS, int ITER, bool LAYER>
__device__ __forceinline__ void normalise(Oct (&v)[ITER], const bool (&live)[ITER], const float* w, const float* b, int col0, const NormParams& p, float* slots) {
    const float inv_n = 1.0f / (float)p.n;
    if (LAYER) {
        uint64_t s = 0;
#pragma unroll
        for (int i = 0; i < ITER; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) s = add_f32x2(s, v[i].v[j]);
        const uint64_t mean = both(-row_sum<THREADS>(sum2(s), slots) * inv_n);
#pragma unroll
        for (int i = 0; i < ITER; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) v[i].v[j] = live[i] ? add_f32x2(v[i].v[j], mean) : 0;
    }
    uint64_t s = 0;
#pragma unroll
    for (int i = 0; i < ITER; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) s = fma_f32x2(v[i].v[j], v[i].v[j], s);
    const uint64_t inv = both(1.0f / sqrtf(row_sum<THREADS>(sum2(s), slots + 32) * inv_n + p.eps));
    const uint64_t offset = both(p.offset);
#pragma unroll
    for (int i = 0; i < ITER; i++) {
        if (live[i]) {
            const int at = col0 + i * THREADS * 8;
#pragma unroll
            for (int j = 0; j < 4; j++) v[i].v[j] = mul_f32x2(v[i].v[j], inv);
            if (w) {
                const Oct t = load8(w + at);
#pragma unroll
                for (int j = 0; j < 4; j++) v[i].v[j] = mul_f32x2(v[i].v[j], add_f32x2(t.v[j], offset));
            }
            if (LAYER && b) {
                const Oct t = load8(b + at);
#pragma unroll
                for (int j = 0; j < 4; j++) v[i].v[j] = add_f32x2(v[i].v[j], t.v[j]);
            }
        }
    }
}

// THREADS threads share a row, each holds ITER pieces of eight elements (piece i of thread t: elements
// 8 * (t + i * THREADS)). THREADS == 32: a warp per row, four rows per CTA; else a CTA per row.
template <int THREADS, int ITER, bool LAYER, bool WIDE>
__global__ void __launch_bounds__(THREADS == 32 ? 128 : THREADS) block_norm_kernel(const NormParams p) {
    __shared__ float slots[4 * 32];
    pdl_launch_dependents();   // the next kernel of the step may be set up beside this one
    pdl_wait();                // the kernel before has completed and its writes are visible
    const int row = THREADS == 32 ? (int)(blockIdx.x * 4 + (threadIdx.x >> 5)) : (int)blockIdx.x;
    const int t = THREADS == 32 ? threadIdx.x & 31 : threadIdx.x;
    if (row >= p.rows) return;                 // whole warps (THREADS == 32); never in the other forms
    const int col0 = 8 * t;
    bool live[ITER];
#pragma unroll
    for (int i = 0; i < ITER; i++) live[i] = col0 + i * THREADS * 8 < p.n;

    Oct h[ITER], b[ITER];
    uint4 raw[ITER][WIDE ? 2 : 1], braw[ITER], graw[ITER];
    const long long grow = p.gate_rows > 0 ? (long long)(row / p.gate_rows) * p.gate_stride : 0;
#pragma unroll
    for (int i = 0; i < ITER; i++) {
        const int at = col0 + i * THREADS * 8;
        raw[i][0] = raw[i][WIDE ? 1 : 0] = braw[i] = graw[i] = make_uint4(0, 0, 0, 0);
        if (live[i]) {
            const char* src = (const char*)p.hidden + ((long long)row * p.hidden_stride + at) * (WIDE ? 4 : 2);
            raw[i][0] = *reinterpret_cast<const uint4*>(src);
            if (WIDE) raw[i][WIDE ? 1 : 0] = *reinterpret_cast<const uint4*>(src + 16);
            if (p.block) braw[i] = *reinterpret_cast<const uint4*>(p.block + (long long)row * p.block_stride + at);
            // a gate in bf16 may be as long as the rows: it travels with them
            if (p.gate_type == OCO_GATE_BF16) graw[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.gate) + grow + at);
        }
    }
    if (p.block) {
#pragma unroll
        for (int i = 0; i < ITER; i++) b[i] = unpack8(braw[i]);
        if (p.post_w) normalise<THREADS, ITER, LAYER>(b, live, p.post_w, p.post_b, col0, p, slots);
        if (p.gate_type) {
#pragma unroll
            for (int i = 0; i < ITER; i++) {
                if (live[i]) {
                    Oct g = p.gate_type == OCO_GATE_F32 ? fetch8(reinterpret_cast<const float*>(p.gate) + grow + col0 + i * THREADS * 8) : unpack8(graw[i]);
                    if (p.gate_act != OCO_GATE_PLAIN) {
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            float lo, hi;
                            f32x2_split(g.v[j], lo, hi);
                            if (p.gate_act == OCO_GATE_SIGMOID) g.v[j] = f32x2(gate_sigmoid(lo), gate_sigmoid(hi));
                            else g.v[j] = f32x2(tanhf(lo), tanhf(hi));
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 4; j++) b[i].v[j] = mul_f32x2(b[i].v[j], g.v[j]);
                }
            }
        }
    }
    const uint64_t rs = both(p.residual_scale), bs = both(p.block_scale);
#pragma unroll
    for (int i = 0; i < ITER; i++) {
        h[i] = WIDE ? pairs8(raw[i][0], raw[i][WIDE ? 1 : 0]) : unpack8(raw[i][0]);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            h[i].v[j] = mul_f32x2(h[i].v[j], rs);
            if (p.block) h[i].v[j] = fma_f32x2(bs, b[i].v[j], h[i].v[j]);
        }
        if (p.hidden_out && live[i]) {
            char* dst = (char*)p.hidden_out + ((long long)row * p.hidden_out_stride + col0 + i * THREADS * 8) * (WIDE ? 4 : 2);
            if (WIDE) {
                *reinterpret_cast<ulonglong2*>(dst) = make_ulonglong2(h[i].v[0], h[i].v[1]);
                *reinterpret_cast<ulonglong2*>(dst + 16) = make_ulonglong2(h[i].v[2], h[i].v[3]);
            } else {
                *reinterpret_cast<uint4*>(dst) = pack8(h[i]);
            }
        }
    }
    if (!p.norm_out) return;
    normalise<THREADS, ITER, LAYER>(h, live, p.pre_w, p.pre_b, col0, p, slots + 64);
#pragma unroll
    for (int i = 0; i < ITER; i++)
        if (live[i]) *reinterpret_cast<uint4*>(p.norm_out + (long long)row * p.norm_out_stride + col0 + i * THREADS * 8) = pack8(h[i]);
}

int say(char* err, size_t len, int code, const char* text) {
    if (err && len) snprintf(err, len, "%s", text);
    return code;
}

// Rows in memory: `count` rows of `width` bytes every `pitch` bytes.
struct Rows {
    uintptr_t at;
    size_t pitch, width, count;
    uintptr_t end() const { return at + (count - 1) * pitch + width; }
};
// Whether two sets of rows share a byte. Interleaved rows of one pitch are told apart; of two pitches they count as shared.
bool overlap(const Rows& a, const Rows& b) {
    if (!a.at || !b.at || a.end() <= b.at || b.end() <= a.at) return false;
    if (a.pitch != b.pitch || a.count == 1 || b.count == 1) return true;
    const size_t d = b.at >= a.at ? (b.at - a.at) % a.pitch : (a.pitch - (a.at - b.at) % a.pitch) % a.pitch;
    return d < a.width || a.pitch - d < b.width;
}

template <int THREADS, int ITER>
cudaError_t launch(const NormParams& p, bool layer, bool wide, cudaStream_t st) {
    const dim3 grid(THREADS == 32 ? (unsigned)((p.rows + 3LL) / 4) : (unsigned)p.rows), block(THREADS == 32 ? 128 : THREADS);
    if (layer) return wide ? launch_dependent(block_norm_kernel<THREADS, ITER, true, true>, grid, block, 0, st, p)
                           : launch_dependent(block_norm_kernel<THREADS, ITER, true, false>, grid, block, 0, st, p);
    return wide ? launch_dependent(block_norm_kernel<THREADS, ITER, false, true>, grid, block, 0, st, p)
                : launch_dependent(block_norm_kernel<THREADS, ITER, false, false>, grid, block, 0, st, p);
}

}  // namespace

extern "C" int oco_moe_block_norm(const oco_moe_block_norm_args* a, int rows, void* cuda_stream, char* err, size_t err_len) {
    if (err && err_len) err[0] = 0;
    if (!a) return OCO_INVALID_ARGUMENT;
    if (a->width < 8 || a->width % 8 || a->width > kMaxWidth) return say(err, err_len, OCO_UNSUPPORTED_SHAPE, "width must be a multiple of 8, 8 .. 32768");
    if (rows < 0) return say(err, err_len, OCO_INVALID_ARGUMENT, "rows must not be negative");
    if (!a->hidden || (!a->hidden_out && !a->norm_out)) return say(err, err_len, OCO_INVALID_ARGUMENT, "hidden and one of hidden_out, norm_out are required");
    if (a->kind != OCO_NORM_RMS && a->kind != OCO_NORM_LAYER) return say(err, err_len, OCO_INVALID_ARGUMENT, "unknown kind of norm");
    if (a->gate_type < OCO_GATE_NONE || a->gate_type > OCO_GATE_F32 || a->gate_act < OCO_GATE_PLAIN || a->gate_act > OCO_GATE_TANH || a->gate_rows < 0)
        return say(err, err_len, OCO_INVALID_ARGUMENT, "unknown gate_type or gate_act, or negative gate_rows");
    if ((a->gate_type != OCO_GATE_NONE) != (a->gate != nullptr)) return say(err, err_len, OCO_INVALID_ARGUMENT, "gate and gate_type do not agree");
    if (!a->block && (a->gate || a->post_w || a->post_b)) return say(err, err_len, OCO_INVALID_ARGUMENT, "a gate or post-norm without a block output");
    if (a->kind == OCO_NORM_RMS && (a->post_b || a->pre_b)) return say(err, err_len, OCO_INVALID_ARGUMENT, "biases belong to the layer norm");
    if ((a->post_b && !a->post_w) || (a->pre_b && !a->pre_w)) return say(err, err_len, OCO_INVALID_ARGUMENT, "a bias without its weight");
    if (!(a->epsilon >= 0.0f)) return say(err, err_len, OCO_INVALID_ARGUMENT, "epsilon must not be negative");
    const void* aligned[] = {a->hidden, a->block, a->post_w, a->post_b, a->pre_w, a->pre_b, a->gate, a->hidden_out, a->norm_out};
    for (const void* q : aligned)
        if ((uintptr_t)q & 15u) return say(err, err_len, OCO_INVALID_ARGUMENT, "pointers must be 16-byte aligned");
    const int64_t strides[] = {a->hidden_stride, a->block_stride, a->gate_stride, a->hidden_out_stride, a->norm_out_stride};
    for (int64_t s : strides)
        if (s != 0 && (s < a->width || s % 8)) return say(err, err_len, OCO_INVALID_ARGUMENT, "strides are multiples of 8 and at least the width (0: the width)");
    if (rows == 0) return OCO_OK;

    NormParams p{};
    auto pitch = [&](int64_t s) { return s ? (long long)s : (long long)a->width; };
    p.hidden = a->hidden; p.block = a->block; p.post_w = a->post_w; p.post_b = a->post_b; p.pre_w = a->pre_w; p.pre_b = a->pre_b;
    p.gate = a->gate; p.hidden_out = a->hidden_out; p.norm_out = a->norm_out;
    p.hidden_stride = pitch(a->hidden_stride); p.block_stride = pitch(a->block_stride); p.gate_stride = pitch(a->gate_stride);
    p.hidden_out_stride = pitch(a->hidden_out_stride); p.norm_out_stride = pitch(a->norm_out_stride);
    p.n = a->width; p.rows = rows; p.gate_type = a->gate_type; p.gate_rows = a->gate_rows; p.gate_act = a->gate_act;
    p.eps = a->epsilon; p.offset = a->weight_offset; p.residual_scale = a->residual_scale; p.block_scale = a->block_scale;
    const bool layer = a->kind == OCO_NORM_LAYER, wide = a->wide != 0;
    const size_t n = (size_t)a->width, es = wide ? 4 : 2, gs = a->gate_type == OCO_GATE_F32 ? 4 : 2, R = (size_t)rows;
    const Rows hidden{(uintptr_t)p.hidden, p.hidden_stride * es, n * es, R}, block{(uintptr_t)p.block, (size_t)p.block_stride * 2, n * 2, R},
        gate{(uintptr_t)p.gate, p.gate_stride * gs, n * gs, p.gate_rows ? (R - 1) / p.gate_rows + 1 : 1}, h_out{(uintptr_t)p.hidden_out, p.hidden_out_stride * es, n * es, R},
        x_out{(uintptr_t)p.norm_out, (size_t)p.norm_out_stride * 2, n * 2, R};
    auto same = [](const Rows& x, const Rows& y) { return x.at == y.at && x.pitch == y.pitch && x.width == y.width; };   // each element is read by its writer
    if ((overlap(h_out, hidden) && !same(h_out, hidden)) || (overlap(x_out, block) && !same(x_out, block)) || overlap(h_out, block) || overlap(x_out, hidden) ||
        overlap(h_out, gate) || overlap(x_out, gate) || overlap(h_out, x_out))
        return say(err, err_len, OCO_INVALID_ARGUMENT, "outputs overlap inputs or each other (hidden_out may be hidden, norm_out may be block)");
    const int pieces = a->width / 8;
    cudaStream_t st = (cudaStream_t)cuda_stream;
    cudaError_t e;
    if (pieces <= 32) e = launch<32, 1>(p, layer, wide, st);
    else if (pieces <= 64) e = launch<32, 2>(p, layer, wide, st);
    else if (pieces <= 128) e = launch<128, 1>(p, layer, wide, st);
    else if (pieces <= 256) e = launch<256, 1>(p, layer, wide, st);
    else if (pieces <= 384) e = launch<192, 2>(p, layer, wide, st);
    else if (pieces <= 512) e = launch<256, 2>(p, layer, wide, st);
    else if (pieces <= 768) e = launch<384, 2>(p, layer, wide, st);
    else if (pieces <= 1024) e = launch<512, 2>(p, layer, wide, st);
    else if (pieces <= 2048) e = launch<1024, 2>(p, layer, wide, st);
    else e = launch<1024, 4>(p, layer, wide, st);
    if (e != cudaSuccess) return say(err, err_len, OCO_CUDA_ERROR, cudaGetErrorString(e));
    return OCO_OK;
}
