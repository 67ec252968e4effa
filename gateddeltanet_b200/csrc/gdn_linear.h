/* What the kernels of the projections share (gdn_linear.cu, gdn_linear_few.cu). */
#ifndef GDN_LINEAR_H
#define GDN_LINEAR_H

#include "gdn_ops.h"
#include "gdn_values.h"

namespace gdn {
namespace ops {

/* x times the normal distribution's function at x. That of -|x| is half of 1 - erf(|x| / sqrt 2), by formula 7.1.26 of
 * Abramowitz and Stegun's Handbook of Mathematical Functions: a polynomial of t = 1 / (1 + 0.3275911 z) times e^(-z^2),
 * off by at most 1.5e-7, so that results are off by at most 7.5e-8 |x| (with their roundings under 4e-7, where
 * half an FP32 step of 4 is 2.4e-7). The library's erff took 30 % more time where this bounds a call. */
__device__ __forceinline__ float gelu(float x) {
    float t, e;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(fabsf(x), 0.3275911f * 0.70710678f, 1.0f)));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * x * (-0.5f * 1.44269504f)));
    float q = fmaf(t, 1.061405429f, -1.453152027f);
    q = fmaf(t, q, 1.421413741f);
    q = fmaf(t, q, -0.284496736f);
    q = fmaf(t, q, 0.254829592f);
    q = 0.5f * t * q * e;
    return x * (x < 0.0f ? q : 1.0f - q);
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
