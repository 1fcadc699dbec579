// The activations of sv2_activation, in fp32.  `EXACT`: the library's expf,
// erff, tanhf and an IEEE divide, a few fp32 ulps in all, for outputs that
// stay in fp32; else exp2 and reciprocal instructions (1 ulp each, the
// exponent's fp32 rounding adds |v| / 2 ulps: below 2^-18 relative wherever
// the result is not far below the 16-bit types' rounding of its inputs).
#pragma once

#include <hip/hip_runtime.h>

#include "seedvr2_hip.h"

namespace sv2
{

constexpr float kActLog2e = 1.4426950408889634f;

// v / (1 + exp(-v))
template <bool EXACT>
__device__ inline float act_silu(float v)
{
    if constexpr (EXACT)
        return v / (1.f + expf(-v));
    else
        return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -kActLog2e));
}

// v/2 (1 + tanh(u)) = v / (1 + exp(-2u)), u = sqrt(2/pi) (v + 0.044715 v^3)
template <bool EXACT>
__device__ inline float act_gelu_tanh(float v)
{
    const float u2 = v * (1.5957691216057308f + 0.07135481282553424f * (v * v));
    if constexpr (EXACT)
        return v / (1.f + expf(-u2));
    else
        return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(u2 * -kActLog2e));
}

// v/2 (1 + erf(v / sqrt(2))) = v/2 erfc(-v / sqrt(2)): the second form keeps
// its relative accuracy where v is large and negative
__device__ inline float act_gelu(float v)
{
    return 0.5f * v * erfcf(v * -0.70710678118654752f);
}

template <int ACT, bool EXACT>
__device__ inline float activate(float v)
{
    if constexpr (ACT == SV2_ACT_SILU)
        return act_silu<EXACT>(v);
    else if constexpr (ACT == SV2_ACT_GELU)
        return act_gelu(v);
    else if constexpr (ACT == SV2_ACT_GELU_TANH)
        return act_gelu_tanh<EXACT>(v);
    else
        return v;
}

} // namespace sv2
