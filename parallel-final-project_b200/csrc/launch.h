// launch.h — kernel launches that report their status as a return value, plain
// or as a programmatic dependent of the previous launch in the stream.
#pragma once

#include <cuda_runtime.h>

#include <tuple>

namespace tqkv {

// Launch through cudaLaunchKernel so the launch status comes back as a return
// value without clearing (or reading) the host thread's pending CUDA error:
// a failed launch stays visible to the caller's next error query, as with
// the reference's <<<...>>> launches.
template <typename... KArgs, typename... Args>
cudaError_t launch_kernel(void (*fn)(KArgs...), dim3 grid, dim3 block, size_t smem,
                          cudaStream_t stream, Args... args) {
    static_assert(sizeof...(KArgs) == sizeof...(Args), "argument count");
    std::tuple<KArgs...> vals(static_cast<KArgs>(args)...);
    void* ptrs[sizeof...(KArgs) > 0 ? sizeof...(KArgs) : 1];
    std::apply([&](auto&... v) {
        int i = 0;
        ((ptrs[i++] = static_cast<void*>(&v)), ...);
    }, vals);
    return cudaLaunchKernel(reinterpret_cast<const void*>(fn), grid, block, ptrs, smem, stream);
}

// Launch as a programmatic dependent of the previous launch in the stream:
// the kernel's CTAs may be dispatched while that launch finishes, and wait
// for it (griddepcontrol.wait) before touching global memory.  Used for the
// decode kernels, whose consecutive launches (one per decode step) otherwise
// leave ~2 us between the end of one and the start of the next.
template <typename... KArgs, typename... Args>
cudaError_t launch_kernel_dependent(void (*fn)(KArgs...), dim3 grid, dim3 block, size_t smem,
                                    cudaStream_t stream, Args... args) {
    static_assert(sizeof...(KArgs) == sizeof...(Args), "argument count");
    std::tuple<KArgs...> vals(static_cast<KArgs>(args)...);
    void* ptrs[sizeof...(KArgs) > 0 ? sizeof...(KArgs) : 1];
    std::apply([&](auto&... v) {
        int i = 0;
        ((ptrs[i++] = static_cast<void*>(&v)), ...);
    }, vals);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(fn), ptrs);
}

}  // namespace tqkv
