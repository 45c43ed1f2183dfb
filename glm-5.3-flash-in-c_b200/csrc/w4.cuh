// w4.cuh - what the kernels of 4-bit products share on the device.
#pragma once

#include "common.cuh"
#include "w4.h"

namespace g5b {

// The clamped SwiGLU (the gate from above only), as the engine's kernels of many rows take it.
__device__ __forceinline__ float swiglu_value(float g, float u, float limit)
{
    g = g > limit ? limit : g;
    u = u > limit ? limit : (u < -limit ? -limit : u);
    return g * sigmoid_near(g) * u;
}

}  // namespace g5b
