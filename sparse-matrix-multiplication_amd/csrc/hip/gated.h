#pragma once
// The activations of gated products: act(g) = g p(g) with
//   silu       p = 1 / (1 + e^-g)
//   gelu       p = Phi(g), the normal distribution's
//   gelu_tanh  p = 1 / (1 + e^(-2 t)), t = sqrt(2 / pi) (g + 0.044715 g^3):
//              (1 + tanh t) / 2
// and act'(g) = p + g p'(g).

#include <hip/hip_runtime.h>

#include "engine.h"

namespace spmm {
namespace engine {
namespace dev {

// 1 / (1 + e^-x) by the hardware's powers of two and reciprocals: off by (|x| + 4) 2^-23
// of itself, which is little beside a 16-bit result's own rounding.
__device__ __forceinline__ float logistic(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504f));
}
constexpr float kTanhScale = 1.59576912f, kTanhCube = 0.044715f;  // 2 sqrt(2 / pi)

__device__ __forceinline__ float gate_share(Act act, float g) {
    if (act == Act::Silu) return logistic(g);
    if (act == Act::Gelu) return 0.5f * erfcf(g * -0.70710678f);
    return logistic(kTanhScale * (g + kTanhCube * g * g * g));
}
// act(g).  -infinity times p = 0 is the limit, 0.
__device__ __forceinline__ float gate_value(Act act, float g) {
    const float lowest = -3.4028235e38f;
    g = g < lowest ? lowest : g;
    return g * gate_share(act, g);
}
// act of eight, the choice made once.
__device__ __forceinline__ void gate_values(Act act, const float (&g)[8], float (&value)[8]) {
    auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) value[i] = f(g[i]);
    };
    if (act == Act::Silu) each([](float x) { return gate_value(Act::Silu, x); });
    else if (act == Act::Gelu) each([](float x) { return gate_value(Act::Gelu, x); });
    else each([](float x) { return gate_value(Act::GeluTanh, x); });
}
// act(g) and act'(g).  Past 128 on either side p' is 0 in fp32, whatever g multiplies it by.
__device__ __forceinline__ void gate_slope(Act act, float g, float& value, float& slope) {
    const float lowest = -3.4028235e38f;
    g = g < lowest ? lowest : g;
    const float p = gate_share(act, g), near = __builtin_amdgcn_fmed3f(g, -128.0f, 128.0f);
    float more;  // p'
    if (act == Act::Gelu) {
        more = 0.39894228f * __builtin_amdgcn_exp2f(near * near * -0.72134752f);
    } else {
        more = p * (1.0f - p);
        if (act == Act::GeluTanh) more *= kTanhScale * (1.0f + 3.0f * kTanhCube * near * near);
    }
    value = g * p;
    slope = p + near * more;
}

}  // namespace dev
}  // namespace engine
}  // namespace spmm
