// Host-side helpers that every translation unit of the library shares: the failure a C entry turns into its status,
// checked CUDA calls, kernel launches, TMA descriptor encoding and per-device kernel attributes.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <set>
#include <string>
#include <utility>

#include "../../include/b200diff.h"

namespace b2d {

// ------------------------------------------------------------ error plumbing
struct Fail {
    b2d_status code;
    std::string msg;
};

[[noreturn]] inline void fail(b2d_status code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    throw Fail{code, buf};
}

#define CK(call)                                                                                   \
    do {                                                                                           \
        cudaError_t e_ = (call);                                                                   \
        if (e_ != cudaSuccess) fail(B2D_ECUDA, "%s failed: %s", #call, cudaGetErrorString(e_));    \
    } while (0)

// ------------------------------------------------------ kernel launches
// Launches inside a PdlScope carry the programmatic-stream-serialization attribute: the next kernel may start
// its prologue (and its constant-weight loads) while this one finishes; every kernel launched this way calls
// pdl_wait before touching data of its predecessors.  Per host thread, so concurrent contexts do not interact.  Set by
// scopes alone: a launch that fails throws, and must not leave it set for the thread's later calls.
inline thread_local bool tl_pdl = false;

struct PdlScope {
    bool prev;
    explicit PdlScope(bool on = true) : prev(tl_pdl) { tl_pdl = on; }
    ~PdlScope() { tl_pdl = prev; }
    PdlScope(const PdlScope&) = delete;
    PdlScope& operator=(const PdlScope&) = delete;
};

template <typename... KArgs, typename... Args>
void launch_k(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, int cluster_x,
              Args&&... args) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    int n = 0;
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    if (cluster_x > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = unsigned(cluster_x);
        attr[n].val.clusterDim.y = 1;
        attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (tl_pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = unsigned(n);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
    if (e != cudaSuccess) fail(B2D_ECUDA, "kernel launch failed: %s", cudaGetErrorString(e));
}

// ---------------------------------------------------------- TMA descriptors
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline std::mutex g_host_mutex;  // guards the process-wide lookups below

inline EncodeTiledFn encode_fn() {
    static std::atomic<EncodeTiledFn> fn{nullptr};
    EncodeTiledFn f = fn.load(std::memory_order_acquire);
    if (!f) {
        std::lock_guard<std::mutex> lock(g_host_mutex);
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        CK(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q));
        if (q != cudaDriverEntryPointSuccess || !p) fail(B2D_ECUDA, "cuTensorMapEncodeTiled unavailable");
        f = reinterpret_cast<EncodeTiledFn>(p);
        fn.store(f, std::memory_order_release);
    }
    return f;
}

// A kernel's dynamic shared-memory limit is an attribute of the function in the CURRENT device's context, so it
// is set once per (kernel, device): a second context on another device in the same process sets its own.
template <typename K>
void set_smem_limit(K* kernel, int bytes) {
    static std::set<std::pair<const void*, int>> done;
    int dev = 0;
    CK(cudaGetDevice(&dev));
    const auto key = std::make_pair(reinterpret_cast<const void*>(kernel), dev);
    std::lock_guard<std::mutex> lock(g_host_mutex);
    if (done.count(key)) return;
    CK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.insert(key);
}

}  // namespace b2d
