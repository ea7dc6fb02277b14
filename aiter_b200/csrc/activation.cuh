// Activations of the fused GEMM epilogue and of the gated activation, on fp32 values.
//
//   relu       x < 0 ? 0 : x                                  (NaN stays)
//   silu       x / (1 + e^-x)
//   gelu       x * Phi(x) = x / 2 * (1 + erf(x / sqrt 2))
//   gelu_tanh  x / 2 * (1 + tanh u), u = sqrt(2 / pi) (x + 0.044715 x^3)  =  x / (1 + e^-2u)
//
// At -inf silu and the gelus give NaN (0 times infinity), as their formulas do.
#pragma once
#include <cuda_runtime.h>

namespace b200 {

enum Activation : int { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_GELU_TANH = 4, ACT_COUNT = 5 };

__device__ __forceinline__ float act_relu(float x) { return x < 0.f ? 0.f : x; }
__device__ __forceinline__ float act_silu(float x) { return __fdividef(x, 1.f + __expf(-x)); }
__device__ __forceinline__ float act_gelu(float x) { return 0.5f * x * (1.f + erff(x * 0.70710678118654752f)); }
__device__ __forceinline__ float act_gelu_tanh(float x)
{
    const float u2 = x * (1.5957691216057308f + 0.071354816272600253f * x * x); // 2 u
    return __fdividef(x, 1.f + __expf(-u2));
}

// One test of `act` for N values (a test per value would sit in every epilogue's innermost loop).
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act)
{
    if(act == ACT_RELU)
    {
#pragma unroll
        for(int i = 0; i < N; ++i)
            v[i] = act_relu(v[i]);
    }
    else if(act == ACT_SILU)
    {
#pragma unroll
        for(int i = 0; i < N; ++i)
            v[i] = act_silu(v[i]);
    }
    else if(act == ACT_GELU)
    {
#pragma unroll
        for(int i = 0; i < N; ++i)
            v[i] = act_gelu(v[i]);
    }
    else if(act == ACT_GELU_TANH)
    {
#pragma unroll
        for(int i = 0; i < N; ++i)
            v[i] = act_gelu_tanh(v[i]);
    }
}

} // namespace b200
