// Host-side helpers of the library's translation units: error text, per-device facts, launches.
#pragma once
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cuda.h>
#include <cuda_runtime.h>
#include <mutex>
#include <utility>

namespace tcbnn {

inline thread_local char g_err[512] = "";

inline int fail(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return 1;
}

#define CUDA_TRY(expr)                                                              \
    do {                                                                            \
        cudaError_t e_ = (expr);                                                    \
        if (e_ != cudaSuccess)                                                      \
            return fail("%s failed: %s", #expr, cudaGetErrorString(e_));            \
    } while (0)

inline int sm_count(int* sms) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return fail("no CUDA device: %s", cudaGetErrorString(e));
    // per-device caches are shared by every host thread that drives a GPU of its own
    static std::atomic<int> cache[64];
    if (dev >= 0 && dev < 64) {
        const int c = cache[dev].load(std::memory_order_relaxed);
        if (c) { *sms = c; return 0; }
    }
    int n = 0;
    e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess || n <= 0) return fail("cannot query SM count: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) cache[dev].store(n, std::memory_order_relaxed);
    *sms = n;
    return 0;
}

// First-use configuration of a kernel on the current device (opt-in shared memory size): done once
// per device, under a lock, because callers may drive several GPUs from threads of one process.
inline std::mutex g_configure_mutex;
template <class F>
int configure_once(bool (&done)[64], F&& configure) {
    int dev = 0;
    cudaGetDevice(&dev);
    std::lock_guard<std::mutex> lock(g_configure_mutex);
    if (dev >= 0 && dev < 64 && done[dev]) return 0;
    const cudaError_t e = configure();
    if (e != cudaSuccess) return fail("cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) done[dev] = true;
    return 0;
}

// Launches `kernel` as a programmatic dependent of whatever precedes it in the stream: its blocks may
// be set up while that still runs, and it waits (griddepcontrol.wait) before it touches anything that
// an earlier launch writes or reads.  Every kernel launched this way executes that wait.
template <class... P, class... A>
cudaError_t launch_dependent_cluster(void (*kernel)(P...), unsigned grid, unsigned cluster, unsigned block, size_t smem, cudaStream_t st, A&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 0 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
}
template <class... P, class... A>
cudaError_t launch_dependent(void (*kernel)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t st, A&&... args) {
    return launch_dependent_cluster(kernel, grid, 0, block, smem, st, std::forward<A>(args)...);
}

inline int launch_check(const char* what) {
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail("%s launch failed: %s", what, cudaGetErrorString(e));
    return 0;
}

using TensorEncode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline TensorEncode tensor_encode() {
    static const TensorEncode encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult r;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) == cudaSuccess && r == cudaDriverEntryPointSuccess
                   ? (TensorEncode)f : (TensorEncode)nullptr;
    }();
    return encode;
}

}  // namespace tcbnn
