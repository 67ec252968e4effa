/* Values of the serving operators' tensors: eight neighbours at a time through
 * 16-byte accesses, or one by one, as FP32. Loads go past L1, where nothing would be
 * found: a CTA reads each value once. What its threads share (a convolution's starts, slots and weights) goes
 * through L1. */
#ifndef GDN_VALUES_H
#define GDN_VALUES_H

#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "gdn_ops.h"

namespace gdn {
namespace ops {

__device__ __forceinline__ float low_bf16(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_bf16(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
    const float4 a = __ldcg(reinterpret_cast<const float4 *>(p)), b = __ldcg(reinterpret_cast<const float4 *>(p) + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void unpack8(const uint4 &w, float (&v)[8]) {
    v[0] = low_bf16(w.x), v[1] = high_bf16(w.x), v[2] = low_bf16(w.y), v[3] = high_bf16(w.y);
    v[4] = low_bf16(w.z), v[5] = high_bf16(w.z), v[6] = low_bf16(w.w), v[7] = high_bf16(w.w);
}
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&v)[8]) {
    unpack8(__ldcg(reinterpret_cast<const uint4 *>(p)), v);
}
__device__ __forceinline__ float load1(const float *p) { return __ldcg(p); }
__device__ __forceinline__ float load1(const __nv_bfloat16 *p) {
    return __uint_as_float((uint32_t)__ldcg(reinterpret_cast<const unsigned short *>(p)) << 16);
}
__device__ __forceinline__ void store8(float *p, const float (&v)[8]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
    return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}
__device__ __forceinline__ void store8(__nv_bfloat16 *p, const float (&v)[8]) { *reinterpret_cast<uint4 *>(p) = pack8(v); }
__device__ __forceinline__ void store4(float *p, float a, float b, float c, float d) { *reinterpret_cast<float4 *>(p) = make_float4(a, b, c, d); }
__device__ __forceinline__ void store4(__nv_bfloat16 *p, float a, float b, float c, float d) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16(a, b), pack_bf16(c, d));
}
__device__ __forceinline__ void store1(float *p, float x) { *p = x; }
__device__ __forceinline__ void store1(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

/* the same of a tensor whose type is known at run time: element i */
__device__ __forceinline__ void load8(const void *p, int64_t i, int type, float (&v)[8]) {
    if (type == kBF16)
        load8(static_cast<const __nv_bfloat16 *>(p) + i, v);
    else
        load8(static_cast<const float *>(p) + i, v);
}
__device__ __forceinline__ float load1(const void *p, int64_t i, int type) {
    return type == kBF16 ? load1(static_cast<const __nv_bfloat16 *>(p) + i) : load1(static_cast<const float *>(p) + i);
}
__device__ __forceinline__ void store8(void *p, int64_t i, int type, const float (&v)[8]) {
    if (type == kBF16)
        store8(static_cast<__nv_bfloat16 *>(p) + i, v);
    else
        store8(static_cast<float *>(p) + i, v);
}
__device__ __forceinline__ void store1(void *p, int64_t i, int type, float x) {
    if (type == kBF16)
        store1(static_cast<__nv_bfloat16 *>(p) + i, x);
    else
        store1(static_cast<float *>(p) + i, x);
}

/* The start of a kernel launched with launch_overlapped: it may run before the kernel before it on the
 * stream has ended. wait_for_previous: until it has, and all that it wrote is visible, to loads of any kind. Every thread
 * that reads or writes global memory calls it first; before it only prefetches to L2, where that kernel's writes go
 * too. let_next_start: the next kernel's CTAs may come as soon as there is room for them. */
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

/* x sigmoid(x) as x / (1 + e^-x) with the approximate instructions for 2^t and 1 / x. What the rounding of t = -x log2 e
 * leaves out of the exponent, -(x + t ln 2), is put back to first order: results are under (9 + |x| / 20) 2^-24 off (2^t
 * 4, the others 5, and the rounding of ln 2), where without it they were 65 2^-24 off at -87 and 16 2^-24 at -15. For
 * x < -87 (results under 1e-36) -0. The exponent is cut at 88 either way, behind which e^-x adds nothing or is all there is:
 * so e is finite, and the correction too. */
__device__ __forceinline__ float silu(float x) {
    const float near = fminf(fmaxf(x, -88.0f), 88.0f), t = near * -1.44269504f;
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    e = fmaf(e, -fmaf(t, 0.693147181f, near), e);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return x * r;
}
/* Without that correction, for results that are rounded to 16 or 8 bits: under (9 + 1.2 |x|) 2^-24, that is 2^-17. 24
 * prompts of 1000 tokens through the convolution take 109 us so and 115 with it, 4096 x 8 gated heads to 8 bits 15.4
 * and 16.0; FP32 results, of more bytes, take as long either way. */
__device__ __forceinline__ float silu_short(float x) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.44269504f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return x * r;
}

/* Two FP32 values as one operand: their products and sums are rounded as by themselves. */
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void split(uint64_t v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
/* silu of both, with the bits of silu() or, if not kLong, of silu_short() */
template <bool kLong>
__device__ __forceinline__ uint64_t silu2(uint64_t x) {
    uint64_t near = x;
    float a, b;
    if (kLong) {
        split(x, a, b);
        near = pair_of(fminf(fmaxf(a, -88.0f), 88.0f), fminf(fmaxf(b, -88.0f), 88.0f));
    }
    const uint64_t t = mul2(near, pair_of(-1.44269504f, -1.44269504f));
    split(t, a, b);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
    uint64_t e = pair_of(a, b);
    if (kLong) e = fma2(e, fma2(t, pair_of(-0.693147181f, -0.693147181f), mul2(near, pair_of(-1.0f, -1.0f))), e);
    split(add2(e, pair_of(1.0f, 1.0f)), a, b);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(b));
    return mul2(x, pair_of(a, b));
}

__host__ __device__ inline bool on16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace ops
}  // namespace gdn

#endif
