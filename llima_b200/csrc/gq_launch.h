// What the launches of the 8-bit float kernels share on the host.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

namespace gq {

// SMs of the current device (at least 2)
inline cudaError_t sm_count(int& sms) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess && sms < 2) e = cudaErrorInvalidDevice;
    return e;
}

// The kernel's shared memory limit, raised once per device and kernel (`done`: a bit per device).
template <class K>
cudaError_t allow_smem(K kern, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    const cudaError_t g = cudaGetDevice(&dev);
    if (g != cudaSuccess) return g;
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
}

// A launch that may begin while the kernel before it on the stream still runs (its kernels call
// after_previous() before they touch memory, so only their set-up overlaps); cluster > 1: in
// clusters of that many CTAs.
template <class... P, class... A>
int launch_early(void (*kern)(P...), unsigned grid, int threads, int smem, cudaStream_t s, unsigned cluster, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
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
    return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, P(args)...));
}

// A function of the loaded driver, or null
template <class F>
F driver_function(const char* name) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint(name, &f, cudaEnableDefault, &r) != cudaSuccess) f = nullptr;
    return reinterpret_cast<F>(f);
}

// Encodes a tensor map; the status as a runtime error code (the driver's have the same numbers).
// The driver wants a context on the calling thread.  Launches bind the device's own, queries do
// not, and a thread whose first CUDA work is one of these calls has none before this.
inline int encode_map(CUtensorMap* map, CUtensorMapDataType type, cuuint32_t rank, const void* p, const cuuint64_t* dims,
                      const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle, CUtensorMapL2promotion l2) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    using GetContext = CUresult (*)(CUcontext*);
    static const Encode encode = driver_function<Encode>("cuTensorMapEncodeTiled");
    static const GetContext context = driver_function<GetContext>("cuCtxGetCurrent");
    if (encode == nullptr || context == nullptr) return static_cast<int>(cudaErrorNotSupported);
    CUcontext c = nullptr;
    if (context(&c) != CUDA_SUCCESS || c == nullptr) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e == cudaSuccess) e = cudaSetDevice(dev);
        if (e != cudaSuccess) return static_cast<int>(e);
    }
    const cuuint32_t step[3] = {1, 1, 1};
    return static_cast<int>(encode(map, type, rank, const_cast<void*>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   swizzle, l2, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE));
}

}  // namespace gq
