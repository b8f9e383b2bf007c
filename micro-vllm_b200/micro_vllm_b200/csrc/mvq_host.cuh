// What the translation units of libmvquant.so share on the host: errors,
// launches and the two product kernels' launchers.
#pragma once

#include "mvquant.h"

#include <cuda_runtime.h>

#include <utility>

#include "w4_linear.cuh"

namespace mvq {

constexpr int kMaxDevices = 64;
constexpr size_t kSmemMost = 227 * 1024;

int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t err, const char* what);

// Programmatic stream serialization (the kernels wait before they read), and a
// cluster along x where one is asked for.
template <typename... Params, typename... Args>
cudaError_t launch(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, int cluster, void* stream,
                   Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

// p as w4_linear.cuh's kernels take it, without the fields that a plan sets.
// `kind`: kF32, kF16, kBF16 or kI8; e4m3 rows are kF16 to the narrow kernel, kE4M3 to the wide one.
int launch_narrow(const LinearParams& p, int kind, int group, bool zeros, int device, int sms, void* stream);
int launch_wide(const LinearParams& p, int kind, int group, bool zeros, int device, int sms, void* stream);

}  // namespace mvq
