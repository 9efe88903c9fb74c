// Products with e4m3 weights and block scales behind oco_moe_f8_* (routed experts) and oco_dense_* (dense products).
#include <algorithm>
#include <new>

#include "f8.cuh"
#include "f8.h"
#include "f8_tiles.cuh"
#include "host.cuh"

using namespace oco;

namespace {
// Rows per tile: the heights of f8_thin_kernel, then f8_wide_kernel's on one SM and on a pair of them. Row maps have boxes
// of as many rows, the pair's two of 128.
constexpr int kTileRows[5] = {16, 32, 64, 128, 256}, kRowBoxes[4] = {16, 32, 64, 128};
constexpr int kWideIndex = 3, kPairIndex = 4;
// Rows up to which a dense product rounds them itself (one launch less; 4 / 8 / 16 rows through 4096 -> 6144 features: 7.5 /
// 9.5 / 13.3 us against 10.1 / 10.2 / 10.3, 8192 -> 1024: 6.9 / 8.5 / 12.0 against 10.1, 2048 -> 512: 5.2 / 5.1 / 5.9 against
// 10), and tokens of a routed call up to which every route is a tile of its own (two launches instead of five; 2048 x 768,
// eight of 128 experts, 1 / 2 / 3 tokens: 17.3 / 21.8 / 25.8 us against 24.7 / 27.6 / 33.4, 4096 x 1536, two of 128: 16.3 /
// 22.6 / 36.4 against 22.3 / 28.1 / 39.7).
constexpr int kOwnRows = 4, kOwnTokens = 3;
enum F8Kind { kF8Projection = OCO_DENSE_PROJECTION, kF8Gated = OCO_DENSE_FFN_SILU_GATE, kF8Experts = 100 };

struct F8Space {
    uint32_t* status = nullptr;
    uint32_t* offsets = nullptr;
    uint32_t* tile_count = nullptr;
    uint32_t* tiles = nullptr;
    uint32_t* route_of_row = nullptr;
    uint32_t* row_of_route = nullptr;
    uint8_t* xq = nullptr;        // codes of the input rows [R][H] (expert-sorted for routed products)
    float* xs = nullptr;          // their scales [H blocks][pitch]
    uint8_t* aq = nullptr;        // codes of the activations [R][F]
    float* as = nullptr;
    float* y = nullptr;           // f32 [R][H], route order
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
    // rows as TMA reads them (boxes of kRowBoxes rows) and the matrices (boxes of 128 rows)
    CUtensorMap map_x[4], map_a[4], map_gate, map_up, map_down;
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
        w.row_of_route = (uint32_t*)take(R * 4);
    }
    w.xq = take(R * H);
    w.xs = (float*)take((H + 127) / 128 * w.pitch * 4);
    if (kind != kF8Projection) {
        w.aq = take(R * F);
        w.as = (float*)take((F + 127) / 128 * w.pitch * 4);
    }
    if (kind == kF8Experts) w.y = (float*)take(R * H * 4);
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

int make_maps(oco_moe_f8_plan* plan) {
    const oco_moe_f8_desc& d = plan->d;
    const uint64_t E = (uint64_t)d.experts, H = (uint64_t)d.hidden, F = (uint64_t)d.ffn;
    if (!encode_tiled()) return plan->fail(OCO_CUDA_ERROR, "cuTensorMapEncodeTiled unavailable");
    CUresult r = encode_rows(&plan->map_up, (void*)plan->w.up_w, E * F, H, 1, 128, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    if (plan->kind != kF8Projection) {
        if (r == CUDA_SUCCESS) r = encode_rows(&plan->map_gate, (void*)plan->w.gate_w, E * F, H, 1, 128, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
        if (r == CUDA_SUCCESS) r = encode_rows(&plan->map_down, (void*)plan->w.down_w, E * H, F, 1, 128, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    }
    return r == CUDA_SUCCESS ? OCO_OK : plan->fail(OCO_CUDA_ERROR, "cuTensorMapEncodeTiled failed (%d)", (int)r);
}

// Rows per tile (index into kTileRows) for `rows` rows of `experts` experts that some row may choose. Many rows: tiles of
// 128 rows on one SM; for a dense product of 1024 rows or more tiles of 256 rows on SM pairs (4096 -> 8192 features, 1024 /
// 2048 / 8192 rows: 39 / 74 / 239 us against 41 / 77 / 251). Experts keep the lower tiles: at 384 rows an expert the second
// half of their last tile is padding too often (gate and up of 64 experts 515 us, in tiles of 256 rows 562).
int tile_index(int rows, int experts) {
    const int avg = (rows + experts - 1) / experts;
    if (experts == 1) return avg <= 16 ? 0 : avg <= 32 ? 1 : avg <= 256 ? 2 : avg < 1024 ? kWideIndex : kPairIndex;
    return avg <= 8 ? 0 : avg <= 20 ? 1 : avg <= 64 ? 2 : kWideIndex;
}

// Parts of the contraction of an f8_thin_kernel item: as many as fill the SMs twice, two blocks of 128 or more each.
unsigned thin_split(const oco_moe_f8_plan* plan, long long items, int blocks) {
    unsigned split = 1;
    while (split < 8 && items * split * 2 <= 2LL * plan->sm_count && blocks >= 4 * (int)split) split *= 2;
    return split;
}

template <int NT, bool GATED, int FORM>
int launch_thin(oco_moe_f8_plan* plan, const F8TileParams& p, const CUtensorMap& rows, const CUtensorMap& w0, const CUtensorMap& w1, int tiles, unsigned split,
                cudaStream_t st) {
    using S = F8Thin<NT, GATED, FORM>;
    auto kernel = f8_thin_kernel<NT, GATED, FORM>;
    OCO_ALLOW_SMEM_ONCE(plan, kernel);
    const int nfeat = (p.n + 127) / 128;
    OCO_CK(plan, launch_dependent_clusters(kernel, split, dim3((unsigned)((long long)tiles * nfeat * split)), dim3(S::kThreads), S::kSmem, st, p, rows, w0, w1));
    plan->launches++;
    return OCO_OK;
}

// One product over the rows of a call. `maps`: the rows' maps by tile height.
template <bool GATED>
int product(oco_moe_f8_plan* plan, const F8TileParams& p, const CUtensorMap* maps, const CUtensorMap& w0, const CUtensorMap& w1, int index, int tiles, int expected,
            cudaStream_t st) {
    const unsigned split = thin_split(plan, (long long)expected * ((p.n + 127) / 128), (p.K + 127) / 128);
    if (index == 0) return launch_thin<16, GATED, kF8Tiles>(plan, p, maps[0], w0, w1, tiles, split, st);
    if (index == 1) return launch_thin<32, GATED, kF8Tiles>(plan, p, maps[1], w0, w1, tiles, split, st);
    if (index == 2) return launch_thin<64, GATED, kF8Tiles>(plan, p, maps[2], w0, w1, tiles, split, st);
    const long long items = (long long)tiles * ((p.n + (GATED ? 127 : 255)) / (GATED ? 128 : 256));
    if (index == kWideIndex) {
        auto kernel = f8_wide_kernel<GATED, false>;
        OCO_ALLOW_SMEM_ONCE(plan, kernel);
        OCO_CK(plan, launch_dependent(kernel, dim3((unsigned)std::min<long long>(items, plan->sm_count)), dim3(F8Wide<false>::kThreads), F8Wide<false>::kSmem, st, p,
                                      maps[kWideIndex], w0, w1));
    } else {
        auto kernel = f8_wide_kernel<GATED, true>;
        OCO_ALLOW_SMEM_ONCE(plan, kernel);
        OCO_CK(plan, launch_dependent_clusters(kernel, 2u, dim3((unsigned)(2 * std::min<long long>(items, plan->sm_count / 2))), dim3(F8Wide<true>::kThreads),
                                               F8Wide<true>::kSmem, st, p, maps[kWideIndex], w0, w1));
    }
    plan->launches++;
    return OCO_OK;
}

// The rows of one call through the plan's products. ids null: dense.
int run_rows(oco_moe_f8_plan* plan, const uint16_t* x, const uint32_t* ids, const float* probs, const uint16_t* residual, uint16_t* out, int rows,
             cudaStream_t st) {
    const oco_moe_f8_desc& d = plan->d;
    F8Space& ws = plan->ws;
    const bool routed = ids != nullptr;
    const int R = rows * d.top_k, H = d.hidden, F = d.ffn, E = d.experts;
    F8TileParams p{};
    p.row_scales = ws.xs; p.pitch = ws.pitch; p.K = H; p.n = F; p.rows = R; p.status = ws.status; p.top_k = d.top_k; p.experts = E;
    // Few rows: the first product rounds them itself, and a few routed tokens need no sorted rows either (a tile per route;
    // the second product sums a token's routes). Both read an expert once per route.
    const int own_tiles = routed ? R : (rows + 15) / 16, nkb = (H + 127) / 128;
    const unsigned own_split = thin_split(plan, (long long)own_tiles * ((F + 127) / 128), nkb);
    if (rows <= (routed ? kOwnTokens : kOwnRows) && (nkb + (int)own_split - 1) / (int)own_split <= F8Thin<16, true, kF8Rows>::kBlocks) {
        p.x = x; p.ids = ids;
        if (plan->kind == kF8Projection) {
            p.s0 = plan->w.up_s; p.out = out;
            return launch_thin<16, false, kF8Rows>(plan, p, plan->map_x[0], plan->map_up, plan->map_up, own_tiles, own_split, st);
        }
        F8TileParams q = p;
        p.s0 = plan->w.gate_s; p.s1 = plan->w.up_s; p.codes = ws.aq; p.code_scales = ws.as;
        if (int rc = launch_thin<16, true, kF8Rows>(plan, p, plan->map_x[0], plan->map_gate, plan->map_up, own_tiles, own_split, st)) return rc;
        q.row_scales = ws.as; q.K = F; q.n = H; q.s0 = plan->w.down_s; q.out = out;
        if (!routed) return product<false>(plan, q, plan->map_a, plan->map_down, plan->map_down, 0, own_tiles, own_tiles, st);
        q.probs = probs; q.residual = residual;
        return launch_thin<16, false, kF8Concat>(plan, q, plan->map_a[0], plan->map_down, plan->map_down, rows,
                                                 thin_split(plan, (long long)rows * ((H + 127) / 128), d.top_k * ((F + 127) / 128)), st);
    }
    const int index = tile_index(R, routed ? std::min(E, R) : 1), nt = kTileRows[index];
    // tiles: exact for a dense product; for routed rows as many as the worst choice of experts makes, and the usual number
    const int tiles = routed ? R / nt + std::min(E, R) : (R + nt - 1) / nt, expected = routed ? std::max(std::min(E, R), R / nt) : tiles;
    if (routed) {
        F8PlanParams pp{ids, ws.offsets, ws.route_of_row, ws.row_of_route, ws.tiles, ws.tile_count, R, E, nt};
        const unsigned ctas = R > 4096 ? 8 : 1;                            // 24576 routes: 28 us on one CTA, 6 on a cluster of eight
        OCO_CK(plan, launch_dependent_clusters(f8_plan_kernel, ctas, dim3(ctas), dim3(1024), 0, st, pp));
        plan->launches++;
    }
    const unsigned row_ctas = (unsigned)(((long long)rows * ((H + 255) / 256) + 15) / 16);
    OCO_CK(plan, launch_dependent(f8_rows_kernel, dim3(row_ctas), dim3(256), 0, st, x, routed ? ws.row_of_route : nullptr, d.top_k, rows, H, ws.xq, ws.xs, ws.pitch));
    plan->launches++;
    if (routed) { p.tiles = ws.tiles; p.tile_count = ws.tile_count; p.offsets = ws.offsets; }
    if (plan->kind == kF8Projection) {
        p.s0 = plan->w.up_s; p.out = out;
        return product<false>(plan, p, plan->map_x, plan->map_up, plan->map_up, index, tiles, expected, st);
    }
    F8TileParams q = p;
    p.s0 = plan->w.gate_s; p.s1 = plan->w.up_s; p.codes = ws.aq; p.code_scales = ws.as;
    if (int rc = product<true>(plan, p, plan->map_x, plan->map_gate, plan->map_up, index, tiles, expected, st)) return rc;
    q.row_scales = ws.as; q.K = F; q.n = H; q.s0 = plan->w.down_s;
    if (routed) { q.sums = ws.y; q.route_of_row = ws.route_of_row; }
    else q.out = out;
    if (int rc = product<false>(plan, q, plan->map_a, plan->map_down, plan->map_down, index, tiles, expected, st)) return rc;
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
    if (plan->weights_device != plan->device)
        return plan->fail(OCO_INVALID_ARGUMENT, "the weights were bound on device %d, the workspace on device %d", plan->weights_device, plan->device);
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
    if (int rc = make_maps(p)) return rc;
    if (int rc = p->note_weights()) return rc;
    OCO_CK(p, cudaDeviceSynchronize());     // calls fetch weights ahead of the work before them: what writes them has ended
    p->have_w = true;
    return OCO_OK;
}

int f8_dense_forward(oco_moe_f8_plan* plan, const uint16_t* x, uint16_t* y, int rows, void* cuda_stream) {
    if (int rc = ready(plan, rows)) return rc;
    if (rows == 0) return OCO_OK;
    if (!x || !y) return plan->fail(OCO_INVALID_ARGUMENT, "null x or y");
    if (((uintptr_t)x | (uintptr_t)y) & 15u) return plan->fail(OCO_INVALID_ARGUMENT, "x and y must be 16-byte aligned");
    const uintptr_t xe = (uintptr_t)x + (size_t)rows * plan->d.hidden * 2, ye = (uintptr_t)y + (size_t)rows * plan->d.ffn * 2;
    if (plan->kind == kF8Projection && (uintptr_t)x < ye && (uintptr_t)y < xe) return plan->fail(OCO_INVALID_ARGUMENT, "y must not overlap x");
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
    // rows, tokens' blocks and pieces of eight columns are counted in 32 bits
    if ((long long)max_rows * plan->d.top_k > (1LL << 28) || (long long)max_rows * plan->d.hidden > (1LL << 33))
        return plan->fail(OCO_UNSUPPORTED_SHAPE, "max_rows * top_k is more than 2^28 or max_rows * hidden more than 2^33");
    if ((uintptr_t)workspace & 255u) return plan->fail(OCO_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
    const F8Space ws = carve(plan->kind, plan->d, max_rows, (unsigned char*)workspace);
    if (bytes < ws.total) return plan->fail(OCO_INVALID_ARGUMENT, "workspace too small: %zu < %zu", bytes, ws.total);
    OCO_CK(plan, cudaDeviceSynchronize());     // whoever had this memory before is done with it
    OCO_CK(plan, cudaMemset(ws.status, 0, 256));
    OCO_CK(plan, cudaDeviceSynchronize());
    if (int rc = plan->note_device()) return rc;
    const uint64_t R = (uint64_t)max_rows * plan->d.top_k;
    if (!encode_tiled()) return plan->fail(OCO_CUDA_ERROR, "cuTensorMapEncodeTiled unavailable");
    for (int i = 0; i < 4; i++) {
        CUresult r = encode_rows(&plan->map_x[i], ws.xq, R, plan->d.hidden, 1, (uint32_t)kRowBoxes[i]);
        if (r == CUDA_SUCCESS && ws.aq) r = encode_rows(&plan->map_a[i], ws.aq, R, plan->d.ffn, 1, (uint32_t)kRowBoxes[i]);
        if (r != CUDA_SUCCESS) return plan->fail(OCO_CUDA_ERROR, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    }
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
    if (int rc = make_maps(plan)) return rc;
    if (int rc = plan->note_weights()) return rc;
    OCO_CK(plan, cudaDeviceSynchronize());  // as in f8_dense_bind_scales
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
    // out = residual: every element is read by its writer
    const size_t bytes = (size_t)rows * plan->d.hidden * 2;
    if (out != residual && (uintptr_t)out < (uintptr_t)residual + bytes && (uintptr_t)residual < (uintptr_t)out + bytes)
        return plan->fail(OCO_INVALID_ARGUMENT, "out must not overlap a part of the residual");
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
