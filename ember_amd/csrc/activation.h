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

// 1 / (1 + e^-x), for x from -87 on within three units in the last place (half steps
// of 2^-24: e^-x 2.7, the sum 1, its reciprocal 2); below, where it is under 2^-125, the
// reciprocal gives 0 for what would not be a normal number.  expf and a division take
// four times as many instructions, which a matrix product's epilogue shows (a gated
// layer of 4096 x 4096 x 8192 in 8 bits: 432 us with them, 419 with this).  e^-x is 2^f *
// 2^n with n whole and f = -x log2(e) - n, |f| <= 1/2, formed with log2(e) in two floats.
// Past +-150 the result is 1 or 0 anyway.
__device__ __forceinline__ float sigmoid(float x)
{
    constexpr float kLog2e = 1.442695041f, kLog2eRest = 1.925963033e-8f;
    x = __builtin_amdgcn_fmed3f(x, -150.0f, 150.0f);
    const float n = __builtin_rintf(x * -kLog2e);
    const float f = __builtin_fmaf(x, -kLog2eRest, __builtin_fmaf(x, -kLog2e, -n));
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f(f), (int)n));
}

// The activations of gated layers: x * sigmoid(c x), with c = 1 SiLU and with c =
// 1.6 Ember's GELU, as (1 + tanh z) / 2 = sigmoid(2 z); c x is rounded, which far below
// 0 is 1.25 |c x| half steps of the result.  An x of -infinity gives NaN, as the formulas
// do, and one with c x below -87 (a result of less than 2^-118) may give -0.
constexpr float kSteepGelu = 1.6f, kSteepSilu = 1.0f;
__device__ __forceinline__ float steepness(int act)
{
    return act == kActGelu ? kSteepGelu : kSteepSilu;
}
// Value and slope.
struct Activated {
    float value, slope;
};
__device__ __forceinline__ Activated activate(float c, float x)
{
    const float s = sigmoid(c * x), v = x * s;
    return {v, s + c * (v * (1.0f - s))};  // c x alone may pass fp32's range
}
// A gated layer's output, and its gradient with respect to both sums.
__device__ __forceinline__ float gated(float c, float gate, float up)
{
    return gate * sigmoid(c * gate) * up;
}
struct GateGrad {
    float gate, up;
};
__device__ __forceinline__ GateGrad gate_grad(float c, float gate, float up, float dh)
{
    const Activated a = activate(c, gate);
    return {dh * up * a.slope, dh * a.value};
}

}  // namespace ember
