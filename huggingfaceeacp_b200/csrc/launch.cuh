// Host-side launch helpers shared by the library's sources.
#pragma once

#include <cuda_runtime.h>

namespace hfk
{
// With `pdl`, the kernel may start before the one ahead of it in the stream has
// ended (it waits with griddepcontrol.wait).
template <typename Kernel, typename... Args>
cudaError_t launch(bool pdl, Kernel kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args)
{
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = block;
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attribute;
    config.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&config, kernel, args...);
}

inline int sm_count(int device)
{
    int sms = 0;
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    return sms > 0 ? sms : 1;
}
} // namespace hfk
