// activation.cuh -- the gate activations of the gated feed-forward product
// and their derivatives, in fp32.
//
// silu and the tanh form of GeLU are both x * sigmoid(y) (0.5 (1 + tanh z) =
// sigmoid(2z)), and sigmoid(y) = 1 / (1 + exp(-y)) loses nothing in the tail,
// where 1 + tanh cancels.  Two special-function operations a value; exp(-y)
// overflows to inf for y below about -88, where the sigmoid is 0 as it should
// be.  The exact GeLU is x Phi(x) with Phi from half_erfc, which keeps the
// tail's relative error as well: two special-function operations too, and the
// polynomial two values at a time (gelu_erf 2048x512x8192 34.4 us, silu 32.0).
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

// Two fp32 multiply-adds as one instruction (sm_100), each rounded like fmaf.
__device__ __forceinline__ float2 fma_pair(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Phi(-|x|) = 0.5 erfc(|x| / sqrt 2) of two values, and e = exp(-x^2 / 2).
// erfc(w) exp(w^2) falls smoothly from 1 to 1 / (w sqrt pi), which
// t = 1 / (1 + p w) follows, so it is t times a polynomial in t, of degree 7,
// fitted to the smallest relative error over 0 <= w <= 10.5, 1.2e-7 (Lawson's
// reweighted least squares at 4000 Chebyshev nodes in t).  With the roundings
// of e's argument the result is good to (8 + 3 x^2 / 2) 2^-24 of its value.  A
// formula of bounded absolute error, such as epilogue.cuh's, is off by 4e-3 of
// the value at x = -4, and a factor U lifts that into H's digits.
__device__ __forceinline__ float2 half_erfc(float2 x, float2& e) {
    auto both = [](float v) { return make_float2(v, v); };
    const float2 w = fma_pair(make_float2(fabsf(x.x), fabsf(x.y)), both(0.23334524f), both(1.0f));
    const float2 t = make_float2(rcp_approx(w.x), rcp_approx(w.y));
    e.x = exp2_approx(x.x * x.x * -0.72134752044448170f);
    e.y = exp2_approx(x.y * x.y * -0.72134752044448170f);
    float2 s = fma_pair(both(-0.0672358455f), t, both(0.228283046f));
    s = fma_pair(s, t, both(-0.172369251f));
    s = fma_pair(s, t, both(0.20123965f));
    s = fma_pair(s, t, both(0.0252482496f));
    s = fma_pair(s, t, both(0.100096691f));
    s = fma_pair(s, t, both(0.0915645922f));
    s = fma_pair(s, t, both(0.0931729062f));
    return make_float2(s.x * t.x * e.x, s.y * t.y * e.y);
}

template <int ACT>
__device__ __forceinline__ float2 act_value2(float2 x) {
    if constexpr (ACT == ACT_SILU) return make_float2(x.x * sigmoid(x.x), x.y * sigmoid(x.y));
    if constexpr (ACT == ACT_GELU_TANH)
        return make_float2(x.x * sigmoid(gelu_tanh_arg(x.x)), x.y * sigmoid(gelu_tanh_arg(x.y)));
    float2 e;
    const float2 q = half_erfc(x, e);
    return make_float2(x.x * (x.x >= 0.f ? 1.0f - q.x : q.x), x.y * (x.y >= 0.f ? 1.0f - q.y : q.y));
}
template <int ACT>
__device__ __forceinline__ float act_value(float x) {
    return act_value2<ACT>(make_float2(x, x)).x;
}

// act(x) and act'(x) together, of two values.  For x sigmoid(y(x)) the derivative is
// p + x p (1 - p) y', with 1 - p = sigmoid(-y).  Where p is 0 the second
// term is 0 too: x and y' stay finite, since y' grows as x^2 and fp16 holds
// |x| <= 65504.  For the exact GeLU it is Phi(x) + x phi(x).
template <int ACT>
__device__ __forceinline__ void act_value_grad2(float2 x, float2& v, float2& d) {
    if constexpr (ACT == ACT_GELU_ERF) {
        float2 e;
        const float2 q = half_erfc(x, e);
        const float2 cdf = make_float2(x.x >= 0.f ? 1.0f - q.x : q.x, x.y >= 0.f ? 1.0f - q.y : q.y);
        v = make_float2(x.x * cdf.x, x.y * cdf.y);
        d = make_float2(fmaf(x.x, 0.3989422804014327f * e.x, cdf.x), fmaf(x.y, 0.3989422804014327f * e.y, cdf.y));
    } else {
        auto one = [](float z, float& value, float& slope) {
            const float y = ACT == ACT_SILU ? z : gelu_tanh_arg(z);
            const float p = sigmoid(y), q = sigmoid(-y);
            value = z * p;
            slope = fmaf(value * q, ACT == ACT_SILU ? 1.0f : gelu_tanh_arg_grad(z), p);
        };
        one(x.x, v.x, d.x);
        one(x.y, v.y, d.y);
    }
}

// The activation chosen at run time (kernels whose time it does not set).
__device__ __forceinline__ float act_value_rt(int act, float x) {
    return act == ACT_SILU ? act_value<ACT_SILU>(x)
                           : act == ACT_GELU_TANH ? act_value<ACT_GELU_TANH>(x) : act_value<ACT_GELU_ERF>(x);
}

}  // namespace pax
