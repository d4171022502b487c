// activation.h -- the activations that kernels apply to sums before they are
// stored (not part of the public ABI).
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>

namespace ember {

// The values of the entry points' `act`.
constexpr int kActNone = 0, kActGelu = 1, kActSilu = 2;

// Ember's GELU, 0.5*x*(1 + tanh(0.8*x)) (ember/nn/activations.py:58), in the
// order Ember's element-wise operators evaluate it.
__device__ __forceinline__ float gelu08(float x)
{
#pragma clang fp contract(off)
    return (x * 0.5f) * (tanhf(x * 0.8f) + 1.0f);
}

// An activation's value and slope.  1 / (1 + e^-x) is 0 where e^-x is infinite,
// and x times it -0: right for every x but -infinity, which gives NaN as the
// formula does.
struct Activated {
    float value, slope;
};
__device__ __forceinline__ Activated activate(int act, float x)
{
    if (act == kActGelu) {
        const float t = tanhf(0.8f * x), half = 0.5f + 0.5f * t;
        return {x * half, half + 0.4f * x * (1.0f - t) * (1.0f + t)};
    }
    const float s = 1.0f / (1.0f + expf(-x));
    return {x * s, s + x * s * (1.0f - s)};
}

// A gated layer's output.
__device__ __forceinline__ float gated(int act, float gate, float up)
{
    return (act == kActGelu ? gelu08(gate) : gate / (1.0f + expf(-gate))) * up;
}

}  // namespace ember
