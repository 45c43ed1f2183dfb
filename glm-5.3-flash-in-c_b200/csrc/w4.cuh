// w4.cuh - what the kernels of 4-bit products share on the device.
#pragma once

#include <cuda.h>

#include "common.cuh"
#include "w4.h"

namespace g5b {

// A tensor map with boxes of any width (tc_stream.cu).
bool tc_encode_swizzled(CUtensorMap *m, const void *base, CUtensorMapDataType dt, int dims, const cuuint64_t *size, const cuuint64_t *stride,
                        const cuuint32_t *box, CUtensorMapSwizzle swizzle);

// The clamped SwiGLU (the gate from above only), as the engine's kernels of many rows take it.
__device__ __forceinline__ float swiglu_value(float g, float u, float limit)
{
    g = g > limit ? limit : g;
    u = u > limit ? limit : (u < -limit ? -limit : u);
    return g * sigmoid_near(g) * u;
}

// The code that a kernel's wait which ran out left in `flag` of the current device (0: none), which is cleared; -1 where it cannot be read.
template <typename FLAG>
inline int w4_flag(FLAG &flag, cudaStream_t st)
{
    int code = 0;
    const int zero = 0;
    if (cudaMemcpyFromSymbolAsync(&code, flag, sizeof code, 0, cudaMemcpyDeviceToHost, st) != cudaSuccess || cudaStreamSynchronize(st) != cudaSuccess) return -1;
    if (code && (cudaMemcpyToSymbolAsync(flag, &zero, sizeof zero, 0, cudaMemcpyHostToDevice, st) != cudaSuccess || cudaStreamSynchronize(st) != cudaSuccess)) return -1;
    return code;
}

}  // namespace g5b
