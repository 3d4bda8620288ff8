// GELU (tanh form) and SiLU as device functors, and their derivatives: shared by the elementwise
// activation and by its checkpointed form.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace hc {

struct ActOp {
    static constexpr bool kBinary = false;
    uint32_t act;  // 0 = GELU (tanh form), 1 = SiLU
    __device__ float apply(float v, float) const {
        if (act == 0) {
            const float kSqrt2OverPi = 0.7978845608f;
            const float kGeluCoeff = 0.044715f;
            float x3 = __fmul_rn(__fmul_rn(v, v), v);
            float inner = __fmul_rn(kSqrt2OverPi, __fadd_rn(v, __fmul_rn(kGeluCoeff, x3)));
            float t = tanhf(inner);
            return __fmul_rn(__fmul_rn(0.5f, v), __fadd_rn(1.0f, t));
        }
        if (v >= 0.0f) {
            float e = expf(-v);
            return __fdiv_rn(v, __fadd_rn(1.0f, e));
        }
        float e = expf(v);
        return __fdiv_rn(__fmul_rn(v, e), __fadd_rn(1.0f, e));
    }
};

// 16-bit outputs: the same functions through the logistic sigmoid, which needs one exponential
// and one reciprocal instead of tanhf / expf / IEEE division:
//   GELU_tanh(x) = 0.5 x (1 + tanh u) = x * sigmoid(2u),  u = sqrt(2/pi) (x + 0.044715 x^3);
//   SiLU(x) = x * sigmoid(x);  sigmoid(z) = 1 / (1 + 2^(-z log2 e)).
// With the constants folded into the base-2 exponent, both are x / (1 + 2^y), y = -x (a + b x^2):
// GELU a = 2 sqrt(2/pi) log2 e, b = 0.044715 a; SiLU a = log2 e, b = 0.  Relative error ~1e-6, far
// below the rounding of the bf16/fp16 result (2^-9 / 2^-12); the fp32 path (ActOp) keeps the
// golden's operation order.  Far below zero 2^y becomes infinite and its reciprocal 0 (from y = 126 on, where it
// would be below the smallest normal number, it is flushed to 0, which takes less than |x| 2^-126 off
// the result): a finite x gives -0 however large it is, as the golden does, and -inf * 0 is NaN, there, too.
// x^2 is held to 256 (at |x| = 16 GELU's y is past 127; SiLU makes no use of it): an infinite one times SiLU's
// b = 0 is NaN.
__device__ __forceinline__ float ex2_ftz(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_ftz(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct FastActOp {
    static constexpr bool kBinary = false;
    float a, b;  // y = -x (a + b x^2)
    __host__ static FastActOp make(uint32_t act) {
        const double log2e = 1.4426950408889634;
        const double k = 2.0 * 0.7978845608028654 * log2e;  // 2 sqrt(2/pi) log2 e
        return act == 0 ? FastActOp{static_cast<float>(k), static_cast<float>(0.044715 * k)}
                        : FastActOp{static_cast<float>(log2e), 0.f};
    }
    __device__ float2 apply2(float2 x) const {
        float2 x2 = __fmul2_rn(x, x);
        x2 = make_float2(fminf(x2.x, 256.f), fminf(x2.y, 256.f));
        const float2 w = __ffma2_rn(make_float2(-b, -b), x2, make_float2(-a, -a));
        const float2 y = __fmul2_rn(x, w);
        const float2 d = __fadd2_rn(make_float2(ex2_ftz(y.x), ex2_ftz(y.y)), make_float2(1.f, 1.f));
        // MUFU rcp: measured faster here than three Newton steps on the FMA pipe
        return __fmul2_rn(x, make_float2(rcp_ftz(d.x), rcp_ftz(d.y)));
    }
    __device__ float apply(float v, float) const { return apply2(make_float2(v, v)).x; }
};

// Slope of either activation at x, with act(x) = x s, s = sigmoid(z(x)):
//   act'(x) = s + x s (1 - s) z'(x)
//   GELU z = 2 sqrt(2/pi) (x + 0.044715 x^3), z' = 2 sqrt(2/pi) (1 + 0.134145 x^2);  SiLU z = x, z' = 1.
// With e = exp(-z) and r = 1 / (1 + e): s = r and 1 - s = e r, so neither side of the sigmoid
// cancels.  Base-2 exponential and hardware reciprocal as in FastActOp, two elements at a time: off by
// some (8 + 3 |z|) half steps of fp32, relative, in either term.  That is far below the rounding of a
// 16-bit gradient and ~2e-7 of an fp32 one, where expf and an IEEE division (~1e-7) made the kernel
// compute-bound (120 us at [16384, 4096] against 92 us of memory time).
// Far out the slope is its limit 0 or 1: x^2 is held to 256, so that x^3 of a huge x does not overflow
// into 0 * inf (beyond |x| = 16, z is long past the fp32 range of the exponential).  The exponent is
// held to 127: there 1 + e is finite and its reciprocal, below the smallest normal number, is flushed
// to 0, and with it the slope, however large x is.  A NaN x stays one through the products with x.
struct ActSlope {
    float a, b;    // z log2 e = x (a + b x^2)
    float za, zb;  // z' = za + zb x^2
    __host__ static ActSlope make(uint32_t act) {
        const double k = 2.0 * 0.7978845608028654, log2e = 1.4426950408889634;
        if (act == 0)
            return ActSlope{static_cast<float>(k * log2e), static_cast<float>(0.044715 * k * log2e),
                            static_cast<float>(k), static_cast<float>(3 * 0.044715 * k)};
        return ActSlope{static_cast<float>(log2e), 0.f, 1.f, 0.f};
    }
    __device__ __forceinline__ float2 apply2(float2 x) const {
        float2 x2 = __fmul2_rn(x, x);
        x2 = make_float2(fminf(x2.x, 256.f), fminf(x2.y, 256.f));
        const float2 y = __fmul2_rn(x, __ffma2_rn(make_float2(-b, -b), x2, make_float2(-a, -a)));
        const float2 e = make_float2(ex2_ftz(fminf(y.x, 127.f)), ex2_ftz(fminf(y.y, 127.f)));
        const float2 d = __fadd2_rn(e, make_float2(1.f, 1.f));
        const float2 r = make_float2(rcp_ftz(d.x), rcp_ftz(d.y));
        const float2 dz = __ffma2_rn(make_float2(zb, zb), x2, make_float2(za, za));
        return __ffma2_rn(__fmul2_rn(__fmul2_rn(x, r), __fmul2_rn(e, r)), dz, r);
    }
    __device__ __forceinline__ float operator()(float x) const { return apply2(make_float2(x, x)).x; }
};

}  // namespace hc
