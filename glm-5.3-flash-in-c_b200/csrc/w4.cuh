// w4.cuh - what the kernels of 4-bit products share on the device.
#pragma once

#include <cuda.h>

#include "common.cuh"
#include "w4.h"

namespace g5b {

// A tensor map with boxes of any width (tc_stream.cu).
bool tc_encode_swizzled(CUtensorMap *m, const void *base, CUtensorMapDataType dt, int dims, const cuuint64_t *size, const cuuint64_t *stride,
                        const cuuint32_t *box, CUtensorMapSwizzle swizzle);

// Eight values from column c on, zero behind the last.
__device__ __forceinline__ void w4_load8(float (&v)[8], const float *row, int c, int cols, bool wide)
{
    if (wide && c + 8 <= cols) {
        const float4 a = *reinterpret_cast<const float4 *>(row + c), b = *reinterpret_cast<const float4 *>(row + c + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = c + i < cols ? row[c + i] : 0.f;
}
__device__ __forceinline__ void w4_load8(float (&v)[8], const uint16_t *row, int c, int cols, bool wide)
{
    if (wide && c + 8 <= cols) {
        const uint4 a = *reinterpret_cast<const uint4 *>(row + c);
        bf16x2_to_f32(a.x, v[0], v[1]); bf16x2_to_f32(a.y, v[2], v[3]); bf16x2_to_f32(a.z, v[4], v[5]); bf16x2_to_f32(a.w, v[6], v[7]);
    } else
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = c + i < cols ? bf16_to_f32(row[c + i]) : 0.f;
}

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
