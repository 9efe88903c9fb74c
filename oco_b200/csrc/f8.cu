// Products with e4m3 weights and block scales behind oco_moe_f8_* (routed experts) and oco_dense_* (dense products).
#include <algorithm>
#include <new>

#include "f8.cuh"
#include "f8.h"
#include "host.cuh"

using namespace oco;

namespace {
enum F8Kind { kF8Projection = OCO_DENSE_PROJECTION, kF8Gated = OCO_DENSE_FFN_SILU_GATE, kF8Experts = 100 };

struct F8Space {
    uint32_t* status = nullptr;
    uint32_t* offsets = nullptr;
    uint32_t* tile_count = nullptr;
    uint32_t* tiles = nullptr;
    uint32_t* route_of_row = nullptr;
    uint8_t* xq = nullptr;        // codes of the input rows [R][H] (expert-sorted for routed products)
    float* xs = nullptr;          // their scales [H blocks][pitch]
    float* act = nullptr;
    uint8_t* aq = nullptr;        // codes of the activations [R][F]
    float* as = nullptr;
    uint16_t* y = nullptr;        // bf16 [R][H], route order
    int pitch = 0;
    size_t total = 0;
};
}  // namespace

struct oco_moe_f8_plan : PlanBase {
    int kind = kF8Experts;
    oco_moe_f8_desc d{};
    oco_moe_f8_weights w{};
    bool have_codes = false;
    F8Space ws{};
};

namespace {

F8Space carve(int kind, const oco_moe_f8_desc& d, int max_rows, unsigned char* base) {
    F8Space w;
    size_t off = 0;
    auto take = [&](size_t bytes) {
        unsigned char* p = base ? base + off : nullptr;
        off = align_up(off + bytes, 256);
        return p;
    };
    const size_t R = (size_t)max_rows * d.top_k, H = (size_t)d.hidden, F = (size_t)d.ffn, E = (size_t)d.experts;
    w.pitch = (int)align_up(R, 128);
    w.status = (uint32_t*)take(256);
    if (kind == kF8Experts) {
        w.offsets = (uint32_t*)take((E + 1) * 4);
        w.tile_count = (uint32_t*)take(4);
        w.tiles = (uint32_t*)take(2 * (R / 16 + std::min(E, R)) * 4);
        w.route_of_row = (uint32_t*)take(R * 4);
    }
    w.xq = take(R * H);
    w.xs = (float*)take((H + 127) / 128 * w.pitch * 4);
    if (kind != kF8Projection) {
        w.act = (float*)take(R * F * 4);
        w.aq = take(R * F);
        w.as = (float*)take((F + 127) / 128 * w.pitch * 4);
    }
    if (kind == kF8Experts) w.y = (uint16_t*)take(R * H * 2);
    w.total = off;
    return w;
}

int check_shape(oco_moe_f8_plan* p) {
    const oco_moe_f8_desc& d = p->d;
    if (d.hidden < 32 || d.hidden % 32 || d.hidden > 65536) return p->fail(OCO_UNSUPPORTED_SHAPE, "hidden must be a multiple of 32, 32 .. 65536");
    if (d.ffn < 32 || d.ffn % 32 || d.ffn > 65536) return p->fail(OCO_UNSUPPORTED_SHAPE, "ffn must be a multiple of 32, 32 .. 65536");
    if (d.experts < 1 || d.experts > kF8MaxExperts) return p->fail(OCO_UNSUPPORTED_SHAPE, "experts must be 1 .. %d", kF8MaxExperts);
    if (d.top_k < 1 || d.top_k > kF8MaxTopK) return p->fail(OCO_UNSUPPORTED_SHAPE, "top_k must be 1 .. %d", kF8MaxTopK);
    return OCO_OK;
}

int check_codes(oco_moe_f8_plan* p) {
    if (!p->w.up_w) return p->fail(OCO_INVALID_ARGUMENT, "up_w is required");
    if (p->kind != kF8Projection && (!p->w.gate_w || !p->w.down_w)) return p->fail(OCO_INVALID_ARGUMENT, "gate_w and down_w are required");
    if (((uintptr_t)p->w.up_w | (uintptr_t)p->w.gate_w | (uintptr_t)p->w.down_w) & 15u) return p->fail(OCO_INVALID_ARGUMENT, "codes must be 16-byte aligned");
    return OCO_OK;
}
int check_scales(oco_moe_f8_plan* p) {
    if (!p->w.up_s) return p->fail(OCO_INVALID_ARGUMENT, "up_s is required");
    if (p->kind != kF8Projection && (!p->w.gate_s || !p->w.down_s)) return p->fail(OCO_INVALID_ARGUMENT, "gate_s and down_s are required");
    if (((uintptr_t)p->w.up_s | (uintptr_t)p->w.gate_s | (uintptr_t)p->w.down_s) & 3u) return p->fail(OCO_INVALID_ARGUMENT, "scales must be 4-byte aligned");
    return OCO_OK;
}

// The rows of one call through the plan's products. ids null: dense.
int run_rows(oco_moe_f8_plan* plan, const uint16_t* x, const uint32_t* ids, const float* probs, const uint16_t* residual, uint16_t* out, int rows,
             cudaStream_t st) {
    const oco_moe_f8_desc& d = plan->d;
    F8Space& ws = plan->ws;
    const bool routed = ids != nullptr;
    const int R = rows * d.top_k, H = d.hidden, F = d.ffn, E = d.experts;
    const uint32_t* live = routed ? ws.offsets + E : nullptr;
    if (routed) {
        F8PlanParams pp{ids, ws.offsets, ws.route_of_row, ws.tiles, ws.tile_count, R, E, 128};
        OCO_CK(plan, launch_dependent(f8_plan_kernel, dim3(1), dim3(1024), 0, st, pp));
        plan->launches++;
    }
    auto grid_for = [&](int k) { return dim3((unsigned)std::min<long long>(((long long)R * ((k + 127) / 128) + 7) / 8, 16LL * plan->sm_count)); };
    OCO_CK(plan, launch_dependent(f8_rows_kernel, grid_for(H), dim3(256), 0, st, x, routed ? ws.route_of_row : nullptr, live, d.top_k, R, H, ws.xq, ws.xs, ws.pitch));
    plan->launches++;
    F8Params p{};
    p.rows = ws.xq; p.row_scales = ws.xs; p.scale_pitch = ws.pitch; p.K = H; p.n = F; p.experts = E; p.dense_rows = R;
    p.offsets = routed ? ws.offsets : nullptr;
    const unsigned row_tiles = (unsigned)std::min(64, (R + 15) / 16);
    if (plan->kind == kF8Projection) {
        p.w0 = plan->w.up_w; p.s0 = plan->w.up_s; p.out = out;
        f8_product_kernel<<<dim3((F + 15) / 16, row_tiles, E), 256, 0, st>>>(p);
        OCO_CK(plan, cudaGetLastError());
        plan->launches++;
        return OCO_OK;
    }
    p.w0 = plan->w.gate_w; p.s0 = plan->w.gate_s; p.w1 = plan->w.up_w; p.s1 = plan->w.up_s; p.act = ws.act;
    f8_product_kernel<<<dim3((F + 15) / 16, row_tiles, E), 256, 0, st>>>(p);
    OCO_CK(plan, cudaGetLastError());
    f8_act_kernel<<<grid_for(F), 256, 0, st>>>(ws.act, live, R, F, ws.aq, ws.as, ws.pitch);
    OCO_CK(plan, cudaGetLastError());
    F8Params q{};
    q.rows = ws.aq; q.row_scales = ws.as; q.scale_pitch = ws.pitch; q.K = F; q.n = H; q.experts = E; q.dense_rows = R;
    q.offsets = p.offsets; q.route_of_row = routed ? ws.route_of_row : nullptr;
    q.w0 = plan->w.down_w; q.s0 = plan->w.down_s; q.out = routed ? ws.y : out;
    f8_product_kernel<<<dim3((H + 15) / 16, row_tiles, E), 256, 0, st>>>(q);
    OCO_CK(plan, cudaGetLastError());
    plan->launches += 3;
    if (routed) {
        const unsigned grid = (unsigned)std::min<long long>(((long long)rows * (H / 8) + 255) / 256, 16LL * plan->sm_count);
        OCO_CK(plan, launch_dependent(f8_combine_kernel, dim3(grid), dim3(256), 0, st, ws.y, ids, probs, residual, out, rows, d.top_k, H, E));
        plan->launches++;
    }
    return OCO_OK;
}

int ready(oco_moe_f8_plan* plan, int rows) {
    plan->launches = 0;
    if (!plan->have_ws || !plan->have_w) return plan->fail(OCO_INVALID_ARGUMENT, "bind a workspace, weights and scales first");
    if (int rc = plan->check_device()) return rc;
    if (rows < 0 || rows > plan->max_rows) return plan->fail(OCO_INVALID_ARGUMENT, "rows %d outside 0..%d", rows, plan->max_rows);
    return OCO_OK;
}

}  // namespace

namespace oco {

int f8_dense_create(const oco_dense_desc& desc, oco_moe_f8_plan** out) {
    oco_moe_f8_plan* p = new (std::nothrow) oco_moe_f8_plan();
    if (!p) return OCO_OUT_OF_MEMORY;
    *out = p;
    p->kind = desc.kind;
    p->d = oco_moe_f8_desc{desc.hidden, desc.ffn, 1, 1};
    if (desc.kind < OCO_DENSE_PROJECTION || desc.kind > OCO_DENSE_FFN_SILU_GATE) return p->fail(OCO_INVALID_ARGUMENT, "unknown dense kind %d", desc.kind);
    if (desc.kind == OCO_DENSE_FFN_RELU2) return p->fail(OCO_UNSUPPORTED_SHAPE, "the relu^2 feed-forward is built for Q4_0 weights");
    return check_shape(p);
}

int f8_dense_bind_codes(oco_moe_f8_plan* p, const oco_dense_weights& w) {
    p->have_codes = p->have_w = false;
    p->w = oco_moe_f8_weights{};
    p->w.up_w = w.up_w;
    if (p->kind == kF8Gated) { p->w.gate_w = w.gate_w; p->w.down_w = w.down_w; }
    if (int rc = check_codes(p)) return rc;
    p->have_codes = true;
    return OCO_OK;
}

int f8_dense_bind_scales(oco_moe_f8_plan* p, const oco_dense_scales& s) {
    p->have_w = false;
    if (!p->have_codes) return p->fail(OCO_INVALID_ARGUMENT, "bind the codes first");
    p->w.up_s = s.up_s;
    if (p->kind == kF8Gated) { p->w.gate_s = s.gate_s; p->w.down_s = s.down_s; }
    if (int rc = check_scales(p)) return rc;
    p->have_w = true;
    return OCO_OK;
}

int f8_dense_forward(oco_moe_f8_plan* plan, const uint16_t* x, uint16_t* y, int rows, void* cuda_stream) {
    if (int rc = ready(plan, rows)) return rc;
    if (rows == 0) return OCO_OK;
    if (!x || !y) return plan->fail(OCO_INVALID_ARGUMENT, "null x or y");
    if (((uintptr_t)x | (uintptr_t)y) & 15u) return plan->fail(OCO_INVALID_ARGUMENT, "x and y must be 16-byte aligned");
    return run_rows(plan, x, nullptr, nullptr, nullptr, y, rows, (cudaStream_t)cuda_stream);
}

}  // namespace oco

extern "C" {

int oco_moe_f8_plan_create(const oco_moe_f8_desc* desc, oco_moe_f8_plan** out) {
    if (!desc || !out) return OCO_INVALID_ARGUMENT;
    oco_moe_f8_plan* p = new (std::nothrow) oco_moe_f8_plan();
    if (!p) return OCO_OUT_OF_MEMORY;
    *out = p;   // handed out even on failure so that the caller can read the message, then destroy
    p->d = *desc;
    return check_shape(p);
}

void oco_moe_f8_plan_destroy(oco_moe_f8_plan* plan) { delete plan; }

size_t oco_moe_f8_workspace_bytes(const oco_moe_f8_plan* plan, int max_rows) {
    return plan && max_rows >= 1 ? carve(plan->kind, plan->d, max_rows, nullptr).total : 0;
}

int oco_moe_f8_bind_workspace(oco_moe_f8_plan* plan, void* workspace, size_t bytes, int max_rows) {
    if (!plan) return OCO_INVALID_ARGUMENT;
    if (!workspace || max_rows < 1) return plan->fail(OCO_INVALID_ARGUMENT, "null workspace or max_rows < 1");
    if ((long long)max_rows * plan->d.top_k > (1LL << 30)) return plan->fail(OCO_UNSUPPORTED_SHAPE, "max_rows * top_k is more than 2^30");
    if ((uintptr_t)workspace & 255u) return plan->fail(OCO_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
    const F8Space ws = carve(plan->kind, plan->d, max_rows, (unsigned char*)workspace);
    if (bytes < ws.total) return plan->fail(OCO_INVALID_ARGUMENT, "workspace too small: %zu < %zu", bytes, ws.total);
    OCO_CK(plan, cudaMemset(ws.status, 0, 256));
    OCO_CK(plan, cudaDeviceSynchronize());
    if (int rc = plan->note_device()) return rc;
    plan->ws = ws;
    plan->max_rows = max_rows;
    plan->have_ws = true;
    return OCO_OK;
}

int oco_moe_f8_bind_weights(oco_moe_f8_plan* plan, const oco_moe_f8_weights* w) {
    if (!plan) return OCO_INVALID_ARGUMENT;
    plan->have_w = false;
    if (!w) return plan->fail(OCO_INVALID_ARGUMENT, "null weights");
    plan->w = *w;
    if (int rc = check_codes(plan)) return rc;
    if (int rc = check_scales(plan)) return rc;
    plan->have_w = true;
    return OCO_OK;
}

int oco_moe_f8_forward(oco_moe_f8_plan* plan, const uint16_t* x, const uint32_t* ids, const float* probs, const uint16_t* residual, uint16_t* out, int rows,
                       void* cuda_stream) {
    if (!plan) return OCO_INVALID_ARGUMENT;
    if (int rc = ready(plan, rows)) return rc;
    if (rows == 0) return OCO_OK;
    if (!x || !ids || !probs || !residual || !out) return plan->fail(OCO_INVALID_ARGUMENT, "null x, ids, probs, residual or out");
    if (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)out) & 15u) return plan->fail(OCO_INVALID_ARGUMENT, "x, residual and out must be 16-byte aligned");
    if (((uintptr_t)ids | (uintptr_t)probs) & 3u) return plan->fail(OCO_INVALID_ARGUMENT, "ids and probs must be 4-byte aligned");
    return run_rows(plan, x, ids, probs, residual, out, rows, (cudaStream_t)cuda_stream);
}

int oco_moe_f8_poll(oco_moe_f8_plan* plan, void* cuda_stream) {
    if (!plan) return OCO_INVALID_ARGUMENT;
    OCO_CK(plan, cudaStreamSynchronize((cudaStream_t)cuda_stream));
    if (!plan->have_ws) return OCO_OK;
    uint32_t word = 0;
    OCO_CK(plan, cudaMemcpy(&word, plan->ws.status, 4, cudaMemcpyDeviceToHost));
    if (!word) return OCO_OK;
    OCO_CK(plan, cudaMemset(plan->ws.status, 0, 4));
    return plan->fail(OCO_DEVICE_TIMEOUT, "a device-side wait gave up");
}

int oco_moe_f8_last_launch_count(const oco_moe_f8_plan* plan) { return plan ? plan->launches : 0; }
const char* oco_moe_f8_last_error(const oco_moe_f8_plan* plan) { return plan ? plan->err : "null plan"; }

}  // extern "C"
