// One way to launch a kernel that may be a programmatic dependent of the kernel ahead of it on the stream, alone or in clusters.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <cstdlib>

namespace ca {

// CA_OPT_DEPENDENT_LAUNCH, as launches carry it
constexpr int DEPENDENT_MERGE = 1, DEPENDENT_ATTENTION = 2;

// dependent: the kernel is set up while the one ahead drains; it executes griddepcontrol.wait before it touches global memory that a kernel may have
// written (work lists that came by copies it may read before).  Where the stream or the driver refuses that (or CA_DISABLE_PDL is
// set), an ordinary launch.  cluster: CTAs of a cluster, along x.
template <typename... P, typename... A>
cudaError_t launch_kernel(void (*kernel)(P...), dim3 grid, int threads, size_t smem, int cluster, bool dependent, cudaStream_t stream, const A&... args) {
    static const bool disabled = std::getenv("CA_DISABLE_PDL") != nullptr;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    const int n = cluster > 1 ? 1 : 0;
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent && !disabled ? n + 1 : n;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e != cudaSuccess && (int)cfg.numAttrs > n) {
        (void)cudaGetLastError();
        cfg.numAttrs = n;
        e = cudaLaunchKernelEx(&cfg, kernel, args...);
    }
    return e;
}

// Once per kernel and device: room for smem bytes of dynamic shared memory, and all of an SM's for it (set at every launch otherwise, for nothing;
// a full table only costs that).
inline cudaError_t allow_shared(const void* kernel, int smem) {
    struct Slot { std::atomic<const void*> kernel{nullptr}; std::atomic<uint64_t> devices{0}; };
    static Slot slots[256];
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    Slot* at = nullptr;
    size_t i = reinterpret_cast<uintptr_t>(kernel) / 16 % 256;
    for (int n = 0; n < 256 && !at; n++, i = (i + 1) % 256) {
        const void* have = slots[i].kernel.load(std::memory_order_relaxed);
        if (have == kernel || (!have && (slots[i].kernel.compare_exchange_strong(have, kernel) || have == kernel))) at = &slots[i];
    }
    const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
    if (at && (at->devices.load(std::memory_order_acquire) & bit)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess && at) at->devices.fetch_or(bit, std::memory_order_release);
    return e;
}

}  // namespace ca
