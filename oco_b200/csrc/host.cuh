// Host-side helpers that the library's translation units share: opt-in shared memory, dependent launches, tensor maps.
#pragma once
#include <atomic>
#include <cstdarg>
#include <cstdio>

#include "common.cuh"

namespace oco {

inline size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

// A kernel's opt-in to large dynamic shared memory is a per-device attribute: this remembers, per
// launch site, on which devices it has been set (bit d = device d). Two threads may both find the
// bit clear and set the attribute twice, which is harmless; a set bit is never lost.
struct DeviceOnce {
    std::atomic<uint64_t> done{0};
    bool need(int dev) const { return dev < 0 || dev >= 64 || !((done.load(std::memory_order_acquire) >> dev) & 1u); }
    void mark(int dev) { if (dev >= 0 && dev < 64) done.fetch_or(1ull << dev, std::memory_order_release); }
};

// Opts a kernel into the full 227 KB of dynamic shared memory; each launch then asks for what it needs.
constexpr size_t kMaxDynamicSmem = 232448;
template <typename Kern>
cudaError_t allow_smem(Kern k) {
    cudaFuncAttributes attr;
    cudaError_t e = cudaFuncGetAttributes(&attr, k);
    if (e != cudaSuccess) return e;
    // static and dynamic shared memory share the 227 KB a CTA may opt into
    return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)(kMaxDynamicSmem - attr.sharedSizeBytes));
}

// Launches a kernel with programmatic stream serialization: it may be scheduled (and, where it does so
// before its griddepcontrol.wait, set up its shared memory and barriers) while its predecessor in the stream
// still runs, and waits for it inside. Every kernel launched this way calls pdl_wait() before it touches
// anything a predecessor wrote or still reads.
template <typename... KArgs, typename... Args>
cudaError_t launch_dependent(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}

// The same for a kernel that runs in clusters of `cluster` CTAs along x.
template <typename... KArgs, typename... Args>
cudaError_t launch_dependent_clusters(void (*kernel)(KArgs...), unsigned cluster, dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                                      Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Looked up once per process (initialisation of a function-local static is thread-safe); null if the driver has none.
inline EncodeTiledFn encode_tiled() {
    static const EncodeTiledFn encode = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            fn = nullptr;
        return (EncodeTiledFn)fn;
    }();
    return encode;
}

// A 2D map over rows of `cols` elements of `elem_bytes` each (1: bytes, 2: 16-bit), box = 128 bytes x box_rows,
// 128-byte swizzle; elements outside read as zero. CUDA_SUCCESS or the driver's answer.
inline CUresult encode_rows(CUtensorMap* map, void* base, uint64_t rows, uint64_t cols, int elem_bytes, uint32_t box_rows,
                            CUtensorMapL2promotion promotion = CU_TENSOR_MAP_L2_PROMOTION_L2_128B) {
    const EncodeTiledFn encode = encode_tiled();
    if (!encode) return CUDA_ERROR_NOT_SUPPORTED;
    cuuint64_t dims[2] = {cols, rows};
    cuuint64_t strides[1] = {cols * (uint64_t)elem_bytes};
    cuuint32_t box[2] = {128u / (uint32_t)elem_bytes, box_rows};
    cuuint32_t estr[2] = {1, 1};
    return encode(map, elem_bytes == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, base, dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, promotion, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// What the plans of the newer entry points have in common: the device their workspace was bound on, the launch
// count of the last call and the last message.
struct PlanBase {
    bool have_ws = false, have_w = false;
    int max_rows = 0, device = -1, weights_device = -1, sm_count = 148, launches = 0;
    char err[256] = {0};

    int fail(int code, const char* fmt, ...) {
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(err, sizeof(err), fmt, ap);
        va_end(ap);
        return code;
    }
    int check_device() {
        int dev = -1;
        if (cudaGetDevice(&dev) != cudaSuccess || dev != device)
            return fail(OCO_INVALID_ARGUMENT, "the plan's workspace was bound on device %d, the current device is %d", device, dev);
        return OCO_OK;
    }
    // The weights that are bound belong to the device that is current then.
    int note_weights() {
        if (cudaGetDevice(&weights_device) != cudaSuccess) return fail(OCO_CUDA_ERROR, "cudaGetDevice failed");
        return OCO_OK;
    }
    int note_device() {
        int dev = 0, sms = 0;
        if (cudaGetDevice(&dev) != cudaSuccess) return fail(OCO_CUDA_ERROR, "cudaGetDevice failed");
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && sms > 0) sm_count = sms;
        device = dev;
        return OCO_OK;
    }
};
#define OCO_CK(plan, call)                                                                                        \
    do {                                                                                                          \
        cudaError_t e_ = (call);                                                                                  \
        if (e_ != cudaSuccess) return (plan)->fail(OCO_CUDA_ERROR, "%s: %s", #call, cudaGetErrorString(e_));      \
    } while (0)
#define OCO_ALLOW_SMEM_ONCE(plan, kernel)                         \
    do {                                                          \
        static oco::DeviceOnce once_;                             \
        if (once_.need((plan)->device)) {                         \
            OCO_CK(plan, oco::allow_smem(kernel));                \
            once_.mark((plan)->device);                           \
        }                                                         \
    } while (0)

}  // namespace oco
