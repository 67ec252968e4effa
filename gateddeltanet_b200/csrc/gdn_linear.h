/* What the kernels of the projections share (gdn_linear.cu, gdn_linear_few.cu). */
#ifndef GDN_LINEAR_H
#define GDN_LINEAR_H

#include "gdn_ops.h"
#include "gdn_values.h"

namespace gdn {
namespace ops {

/* x times the normal distribution's function at x */
__device__ __forceinline__ float gelu(float v) { return 0.5f * v * (1.0f + erff(v * 0.70710678f)); }
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
