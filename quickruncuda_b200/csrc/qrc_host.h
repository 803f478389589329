// qrc_host.h -- host-side helpers shared by the sources of libqrc_b200.so.
#pragma once

#include <cuda_runtime.h>
#include <atomic>
#include <cstdint>
#include <map>
#include <mutex>
#include <new>
#include <utility>

#define QRC_API extern "C" __attribute__((visibility("default")))

// Last CUDA runtime error seen by the library on this thread
// (qrc_last_cuda_error); one variable for all sources.
inline thread_local int g_last_cuda = 0;

#define QRC_CK(call)                                                      \
    do {                                                                  \
        cudaError_t e_ = (call);                                          \
        if (e_ != cudaSuccess) { g_last_cuda = (int)e_; return QRC_ERR_CUDA; } \
    } while (0)

// Makes `dev` current for the scope and restores the caller's device.  When
// `dev` is already current nothing is touched, so a context the caller made
// current through the driver API (as the QuickRunCUDA harness does with
// cuCtxCreate) stays current.
struct DeviceScope {
    int prev = -1;
    bool ok = false, switched = false;
    explicit DeviceScope(int dev) {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (prev == dev) { ok = true; return; }
        ok = cudaSetDevice(dev) == cudaSuccess;
        switched = ok && prev >= 0;
    }
    ~DeviceScope() { if (switched) cudaSetDevice(prev); }
};

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }

// SMs of `dev`, or 0 when there is no such device or it is not an sm_100 one.
// Asked once per device: a device's properties do not change.
inline int sm100_sms(int dev) {
    constexpr int kMaxDevices = 64;
    static std::atomic<int> known[kMaxDevices];
    if (dev < 0 || dev >= kMaxDevices) return 0;
    int sms = known[dev].load(std::memory_order_relaxed);
    if (sms) return sms;
    int ndev = 0, major = 0;
    if (cudaGetDeviceCount(&ndev) != cudaSuccess || dev >= ndev) return 0;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess || major != 10) return 0;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    known[dev].store(sms, std::memory_order_relaxed);
    return sms;
}

// Launches `kernel` with programmatic stream serialization: its CTAs may be
// scheduled while the previous grid in the stream drains.  Only for kernels
// that wait (griddepcontrol.wait) before they touch any memory.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_overlapped(void (*kernel)(KArgs...), dim3 grid, int block, size_t smem, cudaStream_t s,
                                     int cluster, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Raises a kernel's dynamic shared memory limit on the current device to at
// least `smem` (launches above 48 KiB need it).  The attribute is per device,
// so what was granted is remembered per (kernel, device); thread-safe.
inline cudaError_t grant_smem(const void* kernel, size_t smem) {
    if (smem <= 48 * 1024) return cudaSuccess;
    static std::mutex mu;
    static std::map<std::pair<const void*, int>, size_t> granted;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    std::lock_guard<std::mutex> lock(mu);
    try {
        size_t& g = granted[{kernel, dev}];
        if (smem <= g) return cudaSuccess;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e == cudaSuccess) g = smem;
        return e;
    } catch (const std::bad_alloc&) {
        return cudaErrorMemoryAllocation;
    }
}
