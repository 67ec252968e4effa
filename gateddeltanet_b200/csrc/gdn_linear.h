/* What the kernels of the projections share (gdn_linear.cu, gdn_linear_few.cu). */
#ifndef GDN_LINEAR_H
#define GDN_LINEAR_H

#include "gdn_ops.h"
#include "gdn_values.h"

namespace gdn {
namespace ops {

/* x times the normal distribution's function at x. That of -a, a = |x|, is R(a) e^(-a^2 / 2) with R(a) = 0.5 erfcx(a / sqrt 2),
 * which falls smoothly from 0.5 like 1 / a: t = 1 / (1 + c a) times a polynomial of t, fitted to R over a = 0 .. 13.3 for the
 * least relative error (weighted least squares, the weights raised where the error is large, until it is even).
 * The product keeps its relative error where x is far below 0, which 0.5 x (1 + erf(x / sqrt 2)) does not.
 *
 * The polynomial has degree 8 and is off by 2.0e-8; what the roundings of a^2 and of its product leave out of the
 * exponent is put back to first order. In all results are under (20 + a^2 / 40) 2^-24 off: the exponential 4 and its
 * correction 2, the polynomial 2, t 3 (which count up to 2.3 times), the products and 1 - q 5, and the rounding of ln 2. Behind
 * a = 14 the result is x or -0 (of less than 1e-38). Formula 7.1.26 of Abramowitz and Stegun's Handbook, off by 1.5e-7 of
 * 1, was as much as 27 % of the result off at -5; in pairs of values this one takes 3 to 7 % more time where it counts (4096
 * tokens of 512 by 2048 to BF16 18.8 us, 17.5 with the other, to FP32 20.3 and 19.2; one value at a time 29.5). */
__device__ __forceinline__ float gelu(float x) {
    const float a = fminf(fabsf(x), 14.0f), s = a * a, u = s * -0.72134752f;
    float t, e;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(a, 0.345f, 1.0f)));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(u));
    e = fmaf(e, -fmaf(0.5f, fmaf(a, a, -s), fmaf(u, 0.693147181f, 0.5f * s)), e);
    float q = fmaf(t, -0.028427165f, 0.145487756f);
    q = fmaf(t, q, -0.271569431f);
    q = fmaf(t, q, 0.187617302f);
    q = fmaf(t, q, -0.0378698073f);
    q = fmaf(t, q, 0.111904398f);
    q = fmaf(t, q, 0.11721383f);
    q = fmaf(t, q, 0.138023987f);
    q = fmaf(t, q, 0.137619123f);
    q *= t * e;
    return x * (x < 0.0f ? q : 1.0f - q);
}
/* gelu of both, with the bits of gelu() */
__device__ __forceinline__ uint64_t gelu2(uint64_t x) {
    auto both = [](float v) { return pair_of(v, v); };
    float x0, x1, t0, t1, e0, e1;
    split(x, x0, x1);
    const uint64_t a = pair_of(fminf(fabsf(x0), 14.0f), fminf(fabsf(x1), 14.0f)), s = mul2(a, a), u = mul2(s, both(-0.72134752f));
    split(fma2(a, both(0.345f), both(1.0f)), t0, t1);
    split(u, e0, e1);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(t0));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(t1));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e0));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e1));
    const uint64_t t = pair_of(t0, t1), negative = mul2(s, both(-1.0f));
    uint64_t e = pair_of(e0, e1);
    e = fma2(e, fma2(both(-0.5f), fma2(a, a, negative), fma2(u, both(-0.693147181f), mul2(s, both(-0.5f)))), e);
    uint64_t q = fma2(t, both(-0.028427165f), both(0.145487756f));
    q = fma2(t, q, both(-0.271569431f));
    q = fma2(t, q, both(0.187617302f));
    q = fma2(t, q, both(-0.0378698073f));
    q = fma2(t, q, both(0.111904398f));
    q = fma2(t, q, both(0.11721383f));
    q = fma2(t, q, both(0.138023987f));
    q = fma2(t, q, both(0.137619123f));
    q = mul2(q, mul2(t, e));
    float q0, q1, r0, r1;
    split(q, q0, q1);
    split(fma2(q, both(-1.0f), both(1.0f)), r0, r1);
    return mul2(x, pair_of(x0 < 0.0f ? q0 : r0, x1 < 0.0f ? q1 : r1));
}
/* v; `up` is the second half's value for kSwiglu */
__device__ __forceinline__ float activate(int activation, float v, float up) {
    switch (activation) {
        case kSilu: return silu(v);
        case kGelu: return gelu(v);
        case kSwiglu: return silu(v) * up;
        default: return v;
    }
}

}  // namespace ops
}  // namespace gdn

#endif
