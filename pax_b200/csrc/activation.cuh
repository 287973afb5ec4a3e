// activation.cuh -- the gate activations of the gated feed-forward product
// and their derivatives, in fp32.
//
// silu and the tanh form of GeLU are both x * sigmoid(y) (0.5 (1 + tanh z) =
// sigmoid(2z)), and sigmoid(y) = 1 / (1 + exp(-y)) loses nothing in the tail,
// where 1 + tanh cancels.  Two special-function operations a value; exp(-y)
// overflows to inf for y below about -88, where the sigmoid is 0 as it should
// be.  The exact GeLU is epilogue.cuh's gelu_erf (absolute error 3e-7).
#pragma once

#include "epilogue.cuh"

namespace pax {

enum : int { ACT_SILU = 0, ACT_GELU_TANH = 1, ACT_GELU_ERF = 2 };

__device__ __forceinline__ float sigmoid(float y) { return rcp_approx(1.0f + __expf(-y)); }

// 2 z of the tanh form, 2 sqrt(2/pi) (x + 0.044715 x^3), and its derivative.
__device__ __forceinline__ float gelu_tanh_arg(float x) {
    return 1.5957691216057308f * x * fmaf(0.044715f * x, x, 1.0f);
}
__device__ __forceinline__ float gelu_tanh_arg_grad(float x) {
    return 1.5957691216057308f * fmaf(0.134145f * x, x, 1.0f);
}

template <int ACT>
__device__ __forceinline__ float act_value(float x) {
    if constexpr (ACT == ACT_SILU) return x * sigmoid(x);
    if constexpr (ACT == ACT_GELU_TANH) return x * sigmoid(gelu_tanh_arg(x));
    return gelu_erf(x);
}

// act(x) and act'(x) together.  For x sigmoid(y(x)) the derivative is
// p + x p (1 - p) y', with 1 - p = sigmoid(-y).  Where p is 0 the second
// term is 0 too: x and y' stay finite, since y' grows as x^2 and fp16 holds
// |x| <= 65504.  For the exact GeLU it is Phi(x) + x phi(x).
template <int ACT>
__device__ __forceinline__ void act_value_grad(float x, float& v, float& d) {
    if constexpr (ACT == ACT_GELU_ERF) {
        const float q = erfc_hastings(fabsf(x) * 0.70710678118654752f);
        const float cdf = x >= 0.f ? fmaf(-0.5f, q, 1.0f) : 0.5f * q;
        const float phi = 0.3989422804014327f * __expf(-0.5f * x * x);
        v = x * cdf;
        d = fmaf(x, phi, cdf);
    } else {
        const float y = ACT == ACT_SILU ? x : gelu_tanh_arg(x);
        const float p = sigmoid(y), q = sigmoid(-y);
        v = x * p;
        d = fmaf(v * q, ACT == ACT_SILU ? 1.0f : gelu_tanh_arg_grad(x), p);
    }
}

// The activation chosen at run time (kernels whose time it does not set).
__device__ __forceinline__ float act_value_rt(int act, float x) {
    return act == ACT_SILU ? act_value<ACT_SILU>(x)
                           : act == ACT_GELU_TANH ? act_value<ACT_GELU_TANH>(x) : act_value<ACT_GELU_ERF>(x);
}

}  // namespace pax
