// Host pieces every translation unit of the library shares: error state,
// device properties, function attributes and launch helpers. No kernels.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <string>
#include <utility>

#include "../../include/xp_cuda.h"

namespace xp {

inline thread_local std::string g_err;

inline xp_status fail(xp_status s, const char* fmt, ...) {
    char buf[1024];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    g_err = buf;
    return s;
}

#define XP_CUDA_TRY(expr)                                                                          \
    do {                                                                                           \
        cudaError_t e_ = (expr);                                                                   \
        if (e_ != cudaSuccess)                                                                     \
            return ::xp::fail(e_ == cudaErrorMemoryAllocation ? XP_ERR_OOM : XP_ERR_CUDA,          \
                              "%s failed: %s (%s:%d)", #expr, cudaGetErrorString(e_), __FILE__, \
                              __LINE__);                                                           \
    } while (0)

constexpr int kMaxDevices = 64;

inline int sm_count() {
    static std::atomic<int> per_dev[kMaxDevices];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= kMaxDevices) dev = 0;
    int n = per_dev[dev].load(std::memory_order_relaxed);
    if (!n) {
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        if (n <= 0) n = 148;
        per_dev[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

// Function attributes are held per device: raise `kern`'s dynamic shared
// memory limit (and optionally allow non-portable cluster sizes) on the
// current device the first time it launches there. `done` is the call site's
// per-device flag array.
template <typename Kern>
inline cudaError_t smem_attr_once(std::atomic<bool>* done, Kern* kern, int bytes, bool nonportable_cluster = false) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const bool track = dev >= 0 && dev < kMaxDevices;
    if (track && done[dev].load(std::memory_order_acquire)) return cudaSuccess;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && nonportable_cluster)
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && track) done[dev].store(true, std::memory_order_release);
    return e;
}

// Zero-fill device memory and wait for it. cudaMemset runs on the legacy
// default stream, which the library's non-blocking streams do not order
// against: without the wait, a fill could land after the first uploads or
// kernels on those streams. Set-up paths only.
inline cudaError_t zero_fill_sync(void* d, size_t bytes) {
    cudaError_t e = cudaMemset(d, 0, bytes);
    if (e == cudaSuccess) e = cudaStreamSynchronize(cudaStreamLegacy);
    return e;
}
// Host -> device copy that has landed when it returns: a plain cudaMemcpy from
// pageable memory may return once the data is staged, before the DMA that
// work on the non-blocking streams would not wait for. Set-up paths only.
inline cudaError_t h2d_sync(void* dst, const void* src, size_t bytes) {
    cudaError_t e = cudaMemcpy(dst, src, bytes, cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = cudaStreamSynchronize(cudaStreamLegacy);
    return e;
}

// Launch with optional cluster size and programmatic dependent launch.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_ex(void (*k)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                             unsigned cluster_x, bool pdl, Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    unsigned na = 0;
    if (cluster_x > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = cluster_x;
        attr[na].val.clusterDim.y = 1;
        attr[na].val.clusterDim.z = 1;
        ++na;
    }
    if (pdl) {
        attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[na].val.programmaticStreamSerializationAllowed = 1;
        ++na;
    }
    cfg.attrs = attr;
    cfg.numAttrs = na;
    return cudaLaunchKernelEx(&cfg, k, std::forward<Args>(args)...);
}

}  // namespace xp
