/* gdn_norm.cu -- root-mean-square norm of the rows [heads][dim] of a set of
 * tokens, with the additions around it that a layer makes:
 *   h = residual + x (written back to the residual, rounded to its type)
 *   y = h / sqrt(mean(h^2) + eps) * weight * silu(gate)
 *   8 bits: s = max(max |y| / 448, 2^-126) over the token's heads, out = e4m3(y (1 / s))
 * The mean is that of the unrounded sums h, in FP32.
 *
 * Bound by HBM: each value is read and written once. A row is held in
 * registers by a group of threads, sixteen values each, from the loads to the
 * stores; the sum of squares, and the largest value of a token for its scale,
 * are met through shuffles and shared memory in a fixed order. What would cost
 * most is the wait for a row's loads and its two meetings, so each CTA takes
 * rows in turn and the loads of the next one are on their way meanwhile: one
 * row to a CTA without that took 41.6 us where this took 16.4, a ring of rows in
 * shared memory 28.7 where this took 22.5.
 *
 * Measured: 4096 x 2048 BF16 with an FP32 residual, to 8 bits, 17.0 to 17.9 us (5.2 to 5.4
 * TB/s), with a BF16 residual, to BF16, 13.5 us (5.0 TB/s), all FP32 23.4 (5.7), 4096 x 8 gated
 * heads of 256 13.0 to 13.7 us (3.7 TB/s), one row of 2048 1.9 us, which is the launch. Rows of more
 * than 8192 values have 64 registers a thread, spill 150 to 460 bytes and are not fetched ahead: 1024 x
 * 16384 BF16 with a residual 35.0 us (3.8 TB/s), FP32 76.5 (3.5), where 4096 x 8192 BF16 take 49.6 (5.4).
 */
#include <type_traits>

#include "gdn_ops.h"
#include "gdn_values.h"

namespace gdn {
namespace ops {

namespace {

constexpr uint32_t kSmall = 256; /* threads of the CTAs that fetch ahead */

struct NormShape {
    uint32_t group; /* threads of a row: a power of two up to 32, or a multiple of 32 */
    uint32_t rows;  /* rows of a CTA */
    uint32_t token; /* whether a CTA's rows are one token's, whose largest value all of them meet */
};

__device__ __forceinline__ float larger(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
template <bool kMax>
__device__ __forceinline__ float join(float a, float b) {
    return kMax ? larger(a, b) : a + b;
}
/* Over the `group` threads of this thread's row: every one of them gets it.
 * `all` (part of a CTA's threads may have no row): over the whole CTA. */
template <bool kMax, bool kFewWarps>
__device__ __forceinline__ float meet(float v, uint32_t group, bool all, float *partial) {
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (group >= 32 || all) {
#pragma unroll
        for (uint32_t o = 16; o > 0; o >>= 1) v = join<kMax>(v, __shfl_xor_sync(0xffffffffu, v, o));
    } else {
        for (uint32_t o = group / 2; o > 0; o >>= 1) v = join<kMax>(v, __shfl_xor_sync(0xffffffffu, v, o));
    }
    if (all || group > 32) {
        if (lane == 0) partial[warp] = v;
        __syncthreads();
        const uint32_t first = all ? 0 : tid / group * (group / 32), n = all ? blockDim.x / 32 : group / 32;
        if (kFewWarps) {
            v = partial[first];
#pragma unroll
            for (uint32_t i = 1; i < kSmall / 32; ++i)
                if (i < n) v = join<kMax>(v, partial[first + i]);
        } else {
            v = lane < n ? partial[first + lane] : 0.0f;
#pragma unroll
            for (uint32_t o = 16; o > 0; o >>= 1) v = join<kMax>(v, __shfl_xor_sync(0xffffffffu, v, o));
        }
    }
    return v;
}

/* How a thread's eight values lie in a row, `step` values between its pieces:
 *   kEights  neighbours, on 16-byte boundaries (of 8 bits on 8 bytes)
 *   kQuads   two pieces of four, where a row's length or boundaries allow no more
 *   kSingles one by one, for rows off the boundaries of these pieces
 * 4096 rows of 2044 BF16 values and residuals take 15.7 us in pieces of four, 31.0 one by one; of 2048 values with an
 * FP32 residual, to 8 bits, 17.8 by eights, 19.1 by fours. */
enum Layout { kEights, kQuads, kSingles };

/* Eight values as they are in memory: fetched ahead, and FP32 when they are used. */
template <typename T, Layout kLayout>
struct Eight {
    float x[8];
    __device__ __forceinline__ void fetch(const T *p, uint32_t step, uint32_t left) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (uint32_t)j * step < left ? load1(p + j * step) : 0.0f;
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = x[j];
    }
};
template <>
struct Eight<__nv_bfloat16, kEights> {
    uint4 w;
    __device__ __forceinline__ void fetch(const __nv_bfloat16 *p, uint32_t, uint32_t) { w = __ldcg(reinterpret_cast<const uint4 *>(p)); }
    __device__ __forceinline__ void get(float (&v)[8]) const { unpack8(w, v); }
};
template <>
struct Eight<float, kEights> {
    float4 a, b;
    __device__ __forceinline__ void fetch(const float *p, uint32_t, uint32_t) {
        a = __ldcg(reinterpret_cast<const float4 *>(p));
        b = __ldcg(reinterpret_cast<const float4 *>(p) + 1);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
};
template <>
struct Eight<__nv_bfloat16, kQuads> {
    uint2 a, b;
    __device__ __forceinline__ void fetch(const __nv_bfloat16 *p, uint32_t step, uint32_t left) {
        a = __ldcg(reinterpret_cast<const uint2 *>(p));
        b = step < left ? __ldcg(reinterpret_cast<const uint2 *>(p + step)) : make_uint2(0, 0);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const { unpack8(make_uint4(a.x, a.y, b.x, b.y), v); }
};
template <>
struct Eight<float, kQuads> {
    float4 a, b;
    __device__ __forceinline__ void fetch(const float *p, uint32_t step, uint32_t left) {
        a = __ldcg(reinterpret_cast<const float4 *>(p));
        b = step < left ? __ldcg(reinterpret_cast<const float4 *>(p + step)) : make_float4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
};
template <Layout kLayout, typename T>
__device__ __forceinline__ void store_eight(T *p, uint32_t step, uint32_t left, const float (&v)[8]) {
    if constexpr (kLayout == kEights) {
        store8(p, v);
    } else if constexpr (kLayout == kQuads) {
        store4(p, v[0], v[1], v[2], v[3]);
        if (step < left) store4(p + step, v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j * step < left) store1(p + j * step, v[j]);
    }
}

/* T: type of x and gate; R: of the residual. kN: eights of values a thread. kAhead: CTAs of up to kSmall
 * threads, which have the registers to fetch the next row's values while one's meet. */
constexpr int ctas_of(int n) { return n == 1 ? 3 : n == 2 ? 2 : 1; } /* that fit an SM with their registers */
template <typename T, typename R, Layout kLayout, int kN, bool kAhead>
__global__ void __launch_bounds__(kAhead ? kSmall : kMaxNormThreads, kAhead ? ctas_of(kN) : 1) norm_kernel(const __grid_constant__ NormParams p, const NormShape g) {
    __shared__ float partial[2][kMaxNormThreads / 32];
    const uint32_t tid = threadIdx.x, r = tid / g.group, t = tid % g.group, rows = p.tokens * p.heads;
    const uint32_t step = kLayout == kEights ? 8 : kLayout == kQuads ? 4 * g.group : g.group;
    auto at = [&](int i) { return kLayout == kEights ? (i * g.group + t) * 8 : i * 8 * g.group + (kLayout == kQuads ? 4 * t : t); };
    auto left = [&](int i) { return p.dim > at(i) ? p.dim - at(i) : 0u; };
    /* where the j-th of eight is from the first */
    auto apart = [&](int j) { return kLayout == kEights ? (uint32_t)j : kLayout == kQuads ? j / 4 * step + j % 4 : j * step; };

    wait_for_previous();
    let_next_start();
    float w[kN][8];
    if (p.weight != nullptr) {
#pragma unroll
        for (int i = 0; i < kN; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) w[i][j] = 0.0f;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            if (kLayout == kEights) {
                if (left(i)) load8(p.weight, at(i), p.weight_type, w[i]);
            } else if (kLayout == kQuads && p.weight_type == kF32) {
                Eight<float, kQuads> v;
                if (left(i)) v.fetch(static_cast<const float *>(p.weight) + at(i), step, left(i)), v.get(w[i]);
            } else if (kLayout == kQuads) {
                Eight<__nv_bfloat16, kQuads> v;
                if (left(i)) v.fetch(static_cast<const __nv_bfloat16 *>(p.weight) + at(i), step, left(i)), v.get(w[i]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j * step < left(i)) w[i][j] = load1(p.weight, at(i) + j * step, p.weight_type);
            }
        }
    }
    Eight<T, kLayout> x[kN], z[kN];
    Eight<R, kLayout> e[kN];
    const float per_dim = 1.0f / (float)p.dim;
    /* this thread's row, and the step to its next one */
    uint32_t row = blockIdx.x * g.rows + r, token = row / p.heads, head = row - token * p.heads;
    const uint32_t row_step = gridDim.x * g.rows, token_step = row_step / p.heads, head_step = row_step - token_step * p.heads;
    auto fetch = [&]() {
        if (r >= g.rows || row >= rows) return;
        const T *from = static_cast<const T *>(p.x) + token * p.x_token + head * p.x_head;
#pragma unroll
        for (int i = 0; i < kN; ++i)
            if (left(i)) x[i].fetch(from + at(i), step, left(i));
        if (p.residual != nullptr) {
            const R *res = static_cast<const R *>(p.residual) + token * p.residual_token + head * p.residual_head;
#pragma unroll
            for (int i = 0; i < kN; ++i)
                if (left(i)) e[i].fetch(res + at(i), step, left(i));
        }
        if (p.gate != nullptr) {
            const T *gate = static_cast<const T *>(p.gate) + token * p.gate_token + head * p.gate_head;
#pragma unroll
            for (int i = 0; i < kN; ++i)
                if (left(i)) z[i].fetch(gate + at(i), step, left(i));
        }
    };
    if (kAhead) fetch();
    for (uint32_t first = blockIdx.x * g.rows; first < rows; first += row_step) {
        if (!kAhead) fetch();
        const bool live = r < g.rows && row < rows, first_head = head == 0;
        const uint32_t this_token = token;
        const int64_t out = token * p.out_token + head * p.out_head;
        float h[kN][8], gate[kN][8];
#pragma unroll
        for (int i = 0; i < kN; ++i) {
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] = 0.0f;
            if (live && left(i)) x[i].get(h[i]);
        }
        if (p.gate != nullptr) {
#pragma unroll
            for (int i = 0; i < kN; ++i) z[i].get(gate[i]);
        }
        if (p.residual != nullptr && live) {
            R *res = static_cast<R *>(p.residual) + token * p.residual_token + head * p.residual_head;
#pragma unroll
            for (int i = 0; i < kN; ++i)
                if (left(i)) {
                    float v[8];
                    e[i].get(v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[i][j] += v[j];
                    store_eight<kLayout>(res + at(i), step, left(i), h[i]);
                }
        }
        row += row_step, token += token_step, head += head_step;
        if (head >= p.heads) head -= p.heads, ++token;
        if (kAhead) fetch();
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kN; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(h[i][j], h[i][j], sum);
        sum = meet<false, kAhead>(sum, g.group, false, partial[0]);
        /* 1 / sqrt: the instruction's value r after a step of Newton's method, r + r (1 - v r^2) / 2, so that it is off
         * by its rounding. Where squares have overflowed the step makes NaN of r = 0, which would be a row of zeros. */
        const float v = fmaf(sum, per_dim, p.eps), root = rsqrtf(v);
        const float f = fmaf(0.5f * root, fmaf(-v * root, root, 1.0f), root);
#pragma unroll
        for (int i = 0; i < kN; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] *= f;
        if (p.weight != nullptr) {
#pragma unroll
            for (int i = 0; i < kN; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] *= w[i][j];
        }
        /* rows that are not fetched ahead spill, and more with two forms: 1024 x 16384 FP32 86 us, 76 with one */
        if (p.gate != nullptr && (!kAhead || p.out_type == kF32)) {
#pragma unroll
            for (int i = 0; i < kN; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] *= silu(gate[i][j]);
        } else if (kAhead && p.gate != nullptr) {
#pragma unroll
            for (int i = 0; i < kN; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] *= silu_short(gate[i][j]);
        }
        if (p.out_type == kE4M3) {
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < kN; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (live && apart(j) < left(i)) top = larger(top, fabsf(h[i][j]));
            top = meet<true, kAhead>(top, g.group, g.token != 0, partial[1]);
            float scale = top / 448.0f;
            if (scale < 0x1p-126f) scale = 0x1p-126f; /* not for a NaN */
            /* Products with the reciprocal: 4096 x 2048 to 8 bits took 21.2 us with quotients (16.9), and as many values, one in a
             * million, stood one E4M3 step from those of the same formula in plain FP32: by the roundings of y itself. */
            const float inv = 1.0f / scale;
            if (live && t == 0 && first_head) p.scales[this_token] = scale;
            uint8_t *o = static_cast<uint8_t *>(p.out) + out;
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                if (!live || !left(i)) continue;
                if constexpr (kLayout == kSingles) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (j * step < left(i)) o[at(i) + j * step] = __nv_cvt_float_to_fp8(h[i][j] * inv, __NV_SATFINITE, __NV_E4M3);
                } else {
                    uint32_t b[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        b[j] = __nv_cvt_float2_to_fp8x2(make_float2(h[i][2 * j] * inv, h[i][2 * j + 1] * inv), __NV_SATFINITE, __NV_E4M3);
                    const uint2 v = make_uint2(b[0] | (b[1] << 16), b[2] | (b[3] << 16));
                    if constexpr (kLayout == kEights) {
                        *reinterpret_cast<uint2 *>(o + at(i)) = v;
                    } else {
                        *reinterpret_cast<uint32_t *>(o + at(i)) = v.x;
                        if (step < left(i)) *reinterpret_cast<uint32_t *>(o + at(i) + step) = v.y;
                    }
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                if (!live || !left(i)) continue;
                if constexpr (kLayout == kEights)
                    store8(p.out, out + at(i), p.out_type, h[i]);
                else if (p.out_type == kBF16)
                    store_eight<kLayout>(static_cast<__nv_bfloat16 *>(p.out) + out + at(i), step, left(i), h[i]);
                else
                    store_eight<kLayout>(static_cast<float *>(p.out) + out + at(i), step, left(i), h[i]);
            }
        }
        if (g.group > 32 || g.token) __syncthreads(); /* `partial` is free again */
    }
}

template <typename T, typename R, Layout kLayout, int kN, bool kAhead>
cudaError_t launch_norm_t(const NormParams &p, int sms, cudaStream_t stream) {
    NormShape g;
    g.group = norm_group(p.dim, 8 * kN);
    g.token = p.out_type == kE4M3 && p.heads > 1;
    g.rows = g.token ? p.heads : g.group >= 128 ? 1 : 128 / g.group;
    const uint32_t block = (g.group * g.rows + 31) / 32 * 32;
    /* as many CTAs as run at once, each with rows in turn */
    const uint32_t all = (p.tokens * p.heads + g.rows - 1) / g.rows, most = (uint32_t)sms * ((kAhead ? ctas_of(kN) * kSmall : kMaxNormThreads) / block);
    return launch_overlapped(norm_kernel<T, R, kLayout, kN, kAhead>, dim3(all < most ? all : most), block, 0, stream, p, g);
}

/* rows of an operand that all start on a boundary of `values` of its values, of 16 bytes at most */
bool rows_on(uint32_t values, const void *p, int64_t token, int64_t head, const NormParams &n, int type) {
    const int64_t size = type == kF32 ? 4 : type == kBF16 ? 2 : 1, step = size * values < 16 ? size * values : 16;
    return p == nullptr || (reinterpret_cast<uintptr_t>(p) % step == 0 && (n.tokens == 1 || token * size % step == 0) &&
                            (n.heads == 1 || head * size % step == 0));
}

template <typename T>
cudaError_t launch_norm_x(const NormParams &p, int sms, cudaStream_t stream) {
    auto all_on = [&](uint32_t values) {
        return p.dim % values == 0 && rows_on(values, p.x, p.x_token, p.x_head, p, p.type) &&
               rows_on(values, p.gate, p.gate_token, p.gate_head, p, p.type) &&
               rows_on(values, p.residual, p.residual_token, p.residual_head, p, p.residual_type) &&
               rows_on(values, p.out, p.out_token, p.out_head, p, p.out_type);
    };
    const bool weight_on16 = on16(p.weight);
    const int layout = all_on(8) && weight_on16 ? kEights : all_on(4) && weight_on16 ? kQuads : kSingles;
    /* Sixteen values a thread, or thirty-two of long rows; eight where x, residual and results are all FP32, the most bytes.
     * 4096 rows of 2048 with sixteen and with eight: FP32 to BF16 11.0 and 12.0 us, to FP32 13.5 and 14.7, with an FP32
     * residual to 8 bits 19.6 and 23.5, to BF16 20.0 and 19.8, to FP32 25.9 and 23.4 (8192 of 1024 25.7 and 24.8, 16384 of
     * 512 28.1 and 26.2; by fours, 2044, 23.0 either way). One by one eight, for want of registers. Rows too long for 256
     * threads are not fetched ahead. */
    auto pick_as = [&](auto r, auto as) {
        using R = decltype(r);
        constexpr Layout kL = decltype(as)::value;
        if constexpr (kL == kEights && sizeof(T) == 4 && sizeof(R) == 4)
            if (p.residual != nullptr && p.out_type == kF32 && norm_threads(p, 8) <= kSmall) return launch_norm_t<T, R, kL, 1, true>;
        if constexpr (kL != kSingles) {
            if (norm_threads(p, 16) <= kSmall) return launch_norm_t<T, R, kL, 2, true>;
            if (norm_threads(p, 32) <= kSmall) return launch_norm_t<T, R, kL, 4, true>;
        } else if (norm_threads(p, 8) <= kSmall) {
            return launch_norm_t<T, R, kL, 1, true>;
        }
        return norm_threads(p, 8) <= kMaxNormThreads ? launch_norm_t<T, R, kL, 1, false> : launch_norm_t<T, R, kL, 2, false>;
    };
    auto pick = [&](auto r) {
        using R = decltype(r);
        return layout == kEights  ? pick_as(r, std::integral_constant<Layout, kEights>())
               : layout == kQuads ? pick_as(r, std::integral_constant<Layout, kQuads>())
                                  : pick_as(r, std::integral_constant<Layout, kSingles>());
    };
    /* without a residual its type is x's */
    auto *launch = (p.residual != nullptr ? p.residual_type : p.type) == kBF16 ? pick(__nv_bfloat16()) : pick(float());
    return launch(p, sms, stream);
}

}  // namespace

cudaError_t launch_norm(const NormParams &p, int sms, cudaStream_t stream) {
    return p.type == kBF16 ? launch_norm_x<__nv_bfloat16>(p, sms, stream) : launch_norm_x<float>(p, sms, stream);
}

}  // namespace ops
}  // namespace gdn

