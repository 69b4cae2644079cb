#pragma once
// Launch helpers shared by the library's CUDA translation units (defined in
// attention.cu).
#include <cuda_runtime.h>

namespace kvbridge::detail {

// Launch with programmatic stream serialisation (the kernel waits for the
// preceding grid itself). Throws std::runtime_error; honours fail_launch.
void launch_kernel_pdl(const void* fn, dim3 grid, dim3 block, uint32_t smem, cudaStream_t stream,
                       void** args, const char* what);

// The same in clusters of `cluster` consecutive CTAs (at most 8).
void launch_kernel_cluster(const void* fn, dim3 grid, dim3 block, uint32_t cluster, uint32_t smem, cudaStream_t stream,
                           void** args, const char* what);

// SM count of the current device (cached per device).
int device_sms();

}  // namespace kvbridge::detail
