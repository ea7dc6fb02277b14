// Activations of the fused GEMM epilogue and of the gated activation, on fp32 values.
//
//   relu       x < 0 ? 0 : x                                  (NaN stays)
//   silu       x / (1 + e^-x)
//   gelu       x * Phi(x) = x / 2 * (1 + erf(x / sqrt 2))
//   gelu_tanh  x / 2 * (1 + tanh u), u = sqrt(2 / pi) (x + 0.044715 x^3)  =  x / (1 + e^-2u)
//
// At -inf silu and the gelus give NaN (0 times infinity), as their formulas do.
//
// Error as evaluated, relative to the value: silu 2^-21 + |x| 2^-23, gelu 2^-19 + x^2 2^-23, gelu_tanh 2^-21 + |2u| 2^-22.  The first
// term is the approximate reciprocal and power of two and the roundings around them.  The second is the power's argument, rounded to
// 32 bits: it shows far out on the negative side, where the value itself is small (gelu at -5: 1.4e-6 of the value -1.4e-6).  Magnitudes below 2^-119 may
// come out as 0, since both instructions flush (silu below x = -87.3, gelu -13.2, gelu_tanh -10.0).  Carrying the argument in two
// floats would cost two to three instructions a value, and the 16-bit outputs of most calls would not show it.
#pragma once
#include <cuda_runtime.h>

namespace b200 {

enum Activation : int { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_GELU_TANH = 4, ACT_COUNT = 5 };

__device__ __forceinline__ float act_relu(float x) { return x < 0.f ? 0.f : x; }
__device__ __forceinline__ float rcp_approx(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float ex2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two values at a time.  Only gelu's polynomial uses the two-wide fp32 instructions of sm_100: for the short chains of silu and
// gelu_tanh the moves into register pairs cost more than the issue slots they save (6 % of the gated activation's time on
// 16384 x 12288), for gelu they save a little (1 %; in the GEMM's epilogue 39 -> 34 us on 4096 x 4096 x 1024).
__device__ __forceinline__ float2 splat(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 rcp2(float2 x) { return make_float2(rcp_approx(x.x), rcp_approx(x.y)); }
__device__ __forceinline__ float2 ex2_2(float2 x) { return make_float2(ex2_approx(x.x), ex2_approx(x.y)); }
__device__ __forceinline__ float act_silu1(float x) { return x * rcp_approx(1.f + ex2_approx(-1.4426950408889634f * x)); }
__device__ __forceinline__ float2 act_silu(float2 x) { return make_float2(act_silu1(x.x), act_silu1(x.y)); }
// x Phi(x) = max(x, 0) - |x| Phi(-|x|), which cancels nowhere.  Phi(-a) = e^(-a^2 / 2) P(t), t = 1 / (1 + 0.305 a): the form of
// Hastings' approximation of the error function (Abramowitz and Stegun 7.1.26) with eight terms, fitted here by weighted least
// squares; the form's relative error over 0 <= a <= 14.5, in exact arithmetic, is 1e-7 (the roundings come on top, see above).  Behind
// 14.5 the product is below the smallest float.
__device__ __forceinline__ float2 act_gelu(float2 x)
{
    const float2 a = make_float2(fabsf(x.x), fabsf(x.y));
    const float2 t = rcp2(__ffma2_rn(splat(0.305f), a, splat(1.f)));
    const float2 e = ex2_2(__fmul2_rn(__fmul2_rn(x, x), splat(-0.72134752044448170f)));
    float2 p       = splat(0.03663931033810061f);
    p              = __ffma2_rn(p, t, splat(-0.15274771740158233f));
    p              = __ffma2_rn(p, t, splat(0.1853173670582593f));
    p              = __ffma2_rn(p, t, splat(-0.03762262041355916f));
    p              = __ffma2_rn(p, t, splat(0.12084127566747853f));
    p              = __ffma2_rn(p, t, splat(0.10347346698339673f));
    p              = __ffma2_rn(p, t, splat(0.12245871190224042f));
    p              = __ffma2_rn(p, t, splat(0.1216402406951673f));
    const float2 q = __fmul2_rn(__fmul2_rn(a, t), __fmul2_rn(p, e));
    return make_float2(x.x > 15.f ? x.x : fmaxf(x.x, 0.f) - q.x, x.y > 15.f ? x.y : fmaxf(x.y, 0.f) - q.y);
}
__device__ __forceinline__ float act_gelu_tanh1(float x)
{
    const float u = x * fmaf(x * x, -0.10294324f, -2.3022082f); // -2 u log2 e
    return x * rcp_approx(1.f + ex2_approx(u));
}
__device__ __forceinline__ float2 act_gelu_tanh(float2 x) { return make_float2(act_gelu_tanh1(x.x), act_gelu_tanh1(x.y)); }

// One test of `act` for N values, N even or 1 (a test per value would sit in every epilogue's innermost loop).  CLASS: 0 for any
// activation, else only the code of one, 1 standing for none and relu.  (The persistent GEMMs are compiled per class: with all of
// them in one kernel its warps evict one another's instructions.)
template <int CLASS = 0, int N>
__device__ __forceinline__ void activate(float (&v)[N], int act)
{
    constexpr bool any = CLASS == 0;
    if((any || CLASS == 1) && act == ACT_RELU)
    {
#pragma unroll
        for(int i = 0; i < N; ++i)
            v[i] = act_relu(v[i]);
    }
    else if(CLASS == ACT_SILU || (any && act == ACT_SILU))
    {
#pragma unroll
        for(int i = 0; i < N; i += 2)
        {
            const float2 y = act_silu(make_float2(v[i], N > 1 ? v[(i + 1) % N] : 0.f));
            v[i]           = y.x;
            if(N > 1)
                v[(i + 1) % N] = y.y;
        }
    }
    else if(CLASS == ACT_GELU || (any && act == ACT_GELU))
    {
#pragma unroll
        for(int i = 0; i < N; i += 2)
        {
            const float2 y = act_gelu(make_float2(v[i], N > 1 ? v[(i + 1) % N] : 0.f));
            v[i]           = y.x;
            if(N > 1)
                v[(i + 1) % N] = y.y;
        }
    }
    else if(CLASS == ACT_GELU_TANH || (any && act == ACT_GELU_TANH))
    {
#pragma unroll
        for(int i = 0; i < N; i += 2)
        {
            const float2 y = act_gelu_tanh(make_float2(v[i], N > 1 ? v[(i + 1) % N] : 0.f));
            v[i]           = y.x;
            if(N > 1)
                v[(i + 1) % N] = y.y;
        }
    }
}

} // namespace b200
