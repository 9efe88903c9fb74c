// Routing with groups of experts: the router product and the selection (select.cuh) behind oco_moe_router_*.
#include <algorithm>
#include <new>
#include <type_traits>

#include "host.cuh"
#include "router_tiles.cuh"
#include "select.cuh"

using namespace oco;

struct oco_moe_router : PlanBase {
    oco_moe_router_desc d{};
    const float* w = nullptr;
    const float* bias = nullptr;
    uint32_t* status = nullptr;
    uint32_t* arrivals = nullptr;     // route_rows_kernel's counters, left at zero by every call
    float* w_norm = nullptr;          // the largest norms of an expert's weights (SelectParams)
    float* logits = nullptr;
    float* errors = nullptr;          // of the logits of a row, for each 128 experts
    uint16_t* pieces = nullptr;       // the weights as three bf16 pieces [3][experts rounded up to 128][hidden]
    CUtensorMap map_w;
    bool laid_out = false;            // pieces and map match the bound weights and workspace
};

namespace {

int padded(int experts) { return (experts + 127) / 128 * 128; }

struct RouterSpace { size_t status, logits, errors, pieces, total; };
RouterSpace carve(const oco_moe_router_desc& d, int max_rows) {
    RouterSpace s{};
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t at = off; off = align_up(off + bytes, 256); return at; };
    s.status = take(256);
    s.logits = take(d.hidden ? (size_t)max_rows * d.experts * 4 : 0);
    s.errors = take(d.hidden ? (size_t)max_rows * (padded(d.experts) / 128) * 4 : 0);
    s.pieces = take((size_t)3 * padded(d.experts) * d.hidden * 2);
    s.total = off;
    return s;
}

// Lays the weights out for the tensor cores once both they and the workspace are bound.
int lay_out(oco_moe_router* r) {
    r->laid_out = false;
    const oco_moe_router_desc& d = r->d;
    if (!r->have_ws || !r->have_w || !d.hidden) return OCO_OK;
    if (int rc = r->check_device()) return rc;
    if (r->weights_device != r->device)
        return r->fail(OCO_INVALID_ARGUMENT, "the weights were bound on device %d, the workspace on device %d", r->weights_device, r->device);
    const int Ep = padded(d.experts);
    OCO_CK(r, cudaDeviceSynchronize());     // the weights have been written, on whatever stream
    router_pieces_kernel<<<4 * r->sm_count, 256>>>(r->w, r->pieces, d.experts, Ep, d.hidden);
    OCO_CK(r, cudaGetLastError());
    OCO_CK(r, cudaMemset(r->w_norm, 0, 20));
    router_norms_kernel<<<d.experts, 256>>>(r->w, (uint32_t*)r->w_norm, d.hidden);
    OCO_CK(r, cudaGetLastError());
    OCO_CK(r, cudaDeviceSynchronize());
    const CUresult e = encode_rows(&r->map_w, r->pieces, (uint64_t)3 * Ep, (uint64_t)d.hidden, 2, 128, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    if (e != CUDA_SUCCESS) return r->fail(OCO_CUDA_ERROR, "cuTensorMapEncodeTiled failed (%d)", (int)e);
    r->laid_out = true;
    return OCO_OK;
}

// Rows up to which one kernel makes the logits and selects (route_rows_kernel); above, the tensor cores make the logits
// (16 rows, 4096 columns, 256 experts: 11.3 us against 14.8, 1024 columns, 64 experts: 7.1 against 11.3, 8192 columns, 512
// experts 30.4 against 33.5, but 4096 columns, 512 experts 19.8 against 18.0; 24 rows of the first 12.5 against 18.9, of the
// last 25.9 against 20.7).
constexpr int kRowsMax = 16;

// The selection; fused: with the product before it, for few rows.
int launch_select(oco_moe_router* r, const SelectParams& p, bool fused, cudaStream_t st) {
    const int per_lane = (p.E + 31) / 32;
    const dim3 grid = fused ? dim3((p.rows + 3) / 4, (p.E + 7) / 8) : dim3((unsigned)((p.rows + 7LL) / 8)), block(256);
    auto launch = [&](auto width) {
        constexpr int VPL = decltype(width)::value;
        if (fused) return launch_dependent(route_rows_kernel<VPL>, grid, block, 0, st, p, const_cast<float*>(p.logits), r->arrivals);
        return p.x ? launch_dependent(select_kernel<VPL, true>, grid, block, 0, st, p) : launch_dependent(select_kernel<VPL, false>, grid, block, 0, st, p);
    };
    cudaError_t e;
    if (per_lane <= 1) e = launch(std::integral_constant<int, 1>());
    else if (per_lane <= 2) e = launch(std::integral_constant<int, 2>());
    else if (per_lane <= 4) e = launch(std::integral_constant<int, 4>());
    else if (per_lane <= 8) e = launch(std::integral_constant<int, 8>());
    else e = launch(std::integral_constant<int, 16>());
    if (e != cudaSuccess) return r->fail(OCO_CUDA_ERROR, "select: %s", cudaGetErrorString(e));
    r->launches++;
    return OCO_OK;
}

SelectParams select_params(const oco_moe_router* r, const float* logits, int rows, uint32_t* ids, float* probs) {
    const oco_moe_router_desc& d = r->d;
    SelectParams p{};
    p.logits = logits; p.bias = r->bias; p.ids = ids; p.probs = probs; p.status = nullptr;
    p.rows = rows; p.E = d.experts; p.H = d.hidden; p.K = d.top_k; p.G = d.groups; p.TG = d.top_groups; p.best = d.group_best;
    p.score = d.score; p.normalize = d.normalize; p.scale = d.scale;
    return p;
}

}  // namespace

extern "C" {

int oco_moe_router_create(const oco_moe_router_desc* desc, oco_moe_router** out) {
    if (!desc || !out) return OCO_INVALID_ARGUMENT;
    oco_moe_router* r = new (std::nothrow) oco_moe_router();
    if (!r) return OCO_OUT_OF_MEMORY;
    *out = r;   // handed out even on failure so that the caller can read the message, then destroy
    r->d = *desc;
    const oco_moe_router_desc& d = *desc;
    if (d.hidden < 0 || d.hidden > 16384 || d.hidden % 32) return r->fail(OCO_UNSUPPORTED_SHAPE, "hidden must be a multiple of 32, up to 16384 (0: logits only)");
    if (d.experts < 1 || d.experts > kSelMaxExperts) return r->fail(OCO_UNSUPPORTED_SHAPE, "experts must be 1 .. %d", kSelMaxExperts);
    if (d.groups < 1 || d.groups > kSelMaxGroups || d.experts % d.groups) return r->fail(OCO_UNSUPPORTED_SHAPE, "groups must be 1 .. %d and divide the experts", kSelMaxGroups);
    if (d.top_groups < 1 || d.top_groups > d.groups) return r->fail(OCO_INVALID_ARGUMENT, "top_groups must be 1 .. groups");
    if (d.top_k < 1 || d.top_k > kSelMaxTopK) return r->fail(OCO_UNSUPPORTED_SHAPE, "top_k must be 1 .. %d", kSelMaxTopK);
    if (d.top_k > d.top_groups * (d.experts / d.groups)) return r->fail(OCO_INVALID_ARGUMENT, "top_k is more than the experts of top_groups groups");
    if (d.group_best != 1 && d.group_best != 2) return r->fail(OCO_INVALID_ARGUMENT, "group_best must be 1 or 2");
    if (d.score != OCO_SCORE_SIGMOID && d.score != OCO_SCORE_SOFTMAX) return r->fail(OCO_INVALID_ARGUMENT, "unknown score");
    return OCO_OK;
}

void oco_moe_router_destroy(oco_moe_router* r) { delete r; }

size_t oco_moe_router_workspace_bytes(const oco_moe_router* r, int max_rows) { return r && max_rows >= 1 ? carve(r->d, max_rows).total : 0; }

int oco_moe_router_bind_workspace(oco_moe_router* r, void* workspace, size_t bytes, int max_rows) {
    if (!r) return OCO_INVALID_ARGUMENT;
    if (!workspace || max_rows < 1) return r->fail(OCO_INVALID_ARGUMENT, "null workspace or max_rows < 1");
    if ((uintptr_t)workspace & 255u) return r->fail(OCO_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
    if (max_rows > 1 << 28) return r->fail(OCO_UNSUPPORTED_SHAPE, "max_rows is more than 2^28");   // tiles are counted in 32 bits
    const RouterSpace s = carve(r->d, max_rows);
    if (bytes < s.total) return r->fail(OCO_INVALID_ARGUMENT, "workspace too small: %zu < %zu", bytes, s.total);
    OCO_CK(r, cudaDeviceSynchronize());     // whoever had this memory before is done with it
    OCO_CK(r, cudaMemset(workspace, 0, 256));
    OCO_CK(r, cudaDeviceSynchronize());
    if (int rc = r->note_device()) return rc;
    unsigned char* base = (unsigned char*)workspace;
    r->status = (uint32_t*)(base + s.status);
    r->arrivals = r->status + 16;
    r->w_norm = (float*)(r->status + 32);
    r->logits = (float*)(base + s.logits);
    r->errors = (float*)(base + s.errors);
    r->pieces = (uint16_t*)(base + s.pieces);
    r->max_rows = max_rows;
    r->have_ws = true;
    return lay_out(r);
}

int oco_moe_router_bind_weights(oco_moe_router* r, const float* w, const float* bias) {
    if (!r) return OCO_INVALID_ARGUMENT;
    if ((r->d.hidden != 0) != (w != nullptr)) return r->fail(OCO_INVALID_ARGUMENT, "router_w goes with hidden: both or neither");
    if (((uintptr_t)w & 15u) || ((uintptr_t)bias & 3u)) return r->fail(OCO_INVALID_ARGUMENT, "router_w must be 16-byte aligned, bias 4-byte");
    r->have_w = false;
    if (w || bias)
        if (int rc = r->note_weights()) return rc;
    r->w = w; r->bias = bias;
    r->have_w = true;
    return lay_out(r);
}

int oco_moe_router_forward(oco_moe_router* r, const uint16_t* x, int rows, uint32_t* ids, float* probs, float* logits, void* cuda_stream) {
    if (!r) return OCO_INVALID_ARGUMENT;
    r->launches = 0;
    if (!r->d.hidden) return r->fail(OCO_INVALID_ARGUMENT, "this router selects from logits only");
    if (!r->laid_out) return r->fail(OCO_INVALID_ARGUMENT, "bind a workspace and weights first");
    if (int rc = r->check_device()) return rc;
    if (rows < 0 || rows > r->max_rows) return r->fail(OCO_INVALID_ARGUMENT, "rows %d outside 0..%d", rows, r->max_rows);
    if (rows == 0) return OCO_OK;
    if (!x || !ids || !probs) return r->fail(OCO_INVALID_ARGUMENT, "null x, ids or probs");
    if (((uintptr_t)x & 15u) || (((uintptr_t)ids | (uintptr_t)probs | (uintptr_t)logits) & 3u))
        return r->fail(OCO_INVALID_ARGUMENT, "x must be 16-byte aligned; ids, probs and logits 4-byte");
    cudaStream_t st = (cudaStream_t)cuda_stream;
    float* lg = logits ? logits : r->logits;
    const oco_moe_router_desc& d = r->d;
    SelectParams p = select_params(r, lg, rows, ids, probs);
    p.x = x; p.w = r->w; p.status = r->status; p.errors = r->errors; p.w_norm = r->w_norm;
    if (rows > kRowsMax) {
        CUtensorMap map_x;
        const CUresult e = encode_rows(&map_x, (void*)x, (uint64_t)rows, (uint64_t)d.hidden, 2, 128);
        if (e != CUDA_SUCCESS) return r->fail(OCO_CUDA_ERROR, "cuTensorMapEncodeTiled failed (%d)", (int)e);
        OCO_ALLOW_SMEM_ONCE(r, router_tile_kernel);
        const int Ep = padded(d.experts), items = (rows + 127) / 128 * (Ep / 128), chunks = (d.hidden + 63) / 64;
        unsigned split = 1;      // parts of the contraction, four stages of 64 or more each, while they find idle SMs
        while (split < 8 && items * (int)split * 2 <= r->sm_count && chunks >= 8 * (int)split) split *= 2;
        OCO_CK(r, launch_dependent_clusters(router_tile_kernel, split, dim3((unsigned)items * split), dim3(RouterTile::kThreads), RouterTile::kSmem, st, map_x, r->map_w,
                                            lg, r->errors, r->w_norm, rows, d.experts, Ep, d.hidden, r->status));
        r->launches++;
    }
    return launch_select(r, p, rows <= kRowsMax, st);
}

int oco_moe_router_select(oco_moe_router* r, const float* logits, int rows, uint32_t* ids, float* probs, void* cuda_stream) {
    if (!r) return OCO_INVALID_ARGUMENT;
    r->launches = 0;
    if (!r->have_w) return r->fail(OCO_INVALID_ARGUMENT, "bind weights first (NULL for what the plan has not)");
    if (rows < 0) return r->fail(OCO_INVALID_ARGUMENT, "rows must not be negative");
    if (rows == 0) return OCO_OK;
    if (!logits || !ids || !probs) return r->fail(OCO_INVALID_ARGUMENT, "null logits, ids or probs");
    if (((uintptr_t)logits | (uintptr_t)ids | (uintptr_t)probs) & 3u) return r->fail(OCO_INVALID_ARGUMENT, "logits, ids and probs must be 4-byte aligned");
    if (r->bias) {
        int dev = -1;
        if (cudaGetDevice(&dev) != cudaSuccess || dev != r->weights_device)
            return r->fail(OCO_INVALID_ARGUMENT, "the bias was bound on device %d, the current device is %d", r->weights_device, dev);
    }
    return launch_select(r, select_params(r, logits, rows, ids, probs), false, (cudaStream_t)cuda_stream);
}

int oco_moe_router_poll(oco_moe_router* r, void* cuda_stream) {
    if (!r) return OCO_INVALID_ARGUMENT;
    OCO_CK(r, cudaStreamSynchronize((cudaStream_t)cuda_stream));
    if (!r->have_ws) return OCO_OK;
    uint32_t word = 0;
    OCO_CK(r, cudaMemcpy(&word, r->status, 4, cudaMemcpyDeviceToHost));
    if (!word) return OCO_OK;
    OCO_CK(r, cudaMemset(r->status, 0, 4));
    return r->fail(OCO_DEVICE_TIMEOUT, "a device-side wait gave up");
}

int oco_moe_router_last_launch_count(const oco_moe_router* r) { return r ? r->launches : 0; }
const char* oco_moe_router_last_error(const oco_moe_router* r) { return r ? r->err : "null plan"; }

}  // extern "C"
