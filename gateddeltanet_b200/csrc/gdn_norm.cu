/* gdn_norm.cu -- root-mean-square norm of the rows [heads][dim] of a set of
 * tokens, with the additions around it that a layer makes:
 *   h = residual + x (written back to the residual, rounded to its type)
 *   y = h / sqrt(mean(h^2) + eps) * weight * silu(gate)
 *   8 bits: s = max(max |y| / 448, 2^-126) over the token's heads, out = e4m3(y / s)
 * The mean is that of the unrounded sums h, in FP32.
 *
 * Bound by HBM: each value is read and written once. A row is held in
 * registers by a group of threads, eight values (or sixteen) each, from the
 * loads to the stores; the sum of squares, and the largest value of a token
 * for its scale, are met through shuffles and shared memory in a fixed order.
 */
#include "gdn_ops.h"
#include "gdn_values.h"

namespace gdn {
namespace ops {

namespace {

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
template <bool kMax>
__device__ __forceinline__ float meet(float v, uint32_t group, bool all, float *partial) {
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t width = all || group > 32 ? 32 : group;
    for (uint32_t o = width / 2; o > 0; o >>= 1) v = join<kMax>(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (width == 32 && (all || group > 32)) {
        if (lane == 0) partial[warp] = v;
        __syncthreads();
        const uint32_t first = all ? 0 : tid / group * (group / 32), n = all ? blockDim.x / 32 : group / 32;
        v = lane < n ? partial[first + lane] : 0.0f;
        for (uint32_t o = 16; o > 0; o >>= 1) v = join<kMax>(v, __shfl_xor_sync(0xffffffffu, v, o));
    }
    return v;
}

/* T: type of x and gate. kWide: eight neighbours to a vector, all rows on
 * 16-byte boundaries; else values `group` apart. kN: eights of values a thread. */
template <typename T, bool kWide, int kN>
__global__ void __launch_bounds__(kMaxNormThreads) norm_kernel(const __grid_constant__ NormParams p, const NormShape g) {
    __shared__ float partial[2][kMaxNormThreads / 32];
    const uint32_t tid = threadIdx.x, r = tid / g.group, t = tid % g.group;
    const uint64_t row = (uint64_t)blockIdx.x * g.rows + r;
    const uint32_t token = (uint32_t)(row / p.heads), head = (uint32_t)(row % p.heads);
    const bool live = r < g.rows && row < (uint64_t)p.tokens * p.heads;
    const uint32_t D = live ? p.dim : 0;
    const T *x = static_cast<const T *>(p.x) + token * p.x_token + head * p.x_head;
    const T *gate = static_cast<const T *>(p.gate) + token * p.gate_token + head * p.gate_head;
    const int64_t res = token * p.residual_token + head * p.residual_head;
    auto at = [&](int i, int j) { return kWide ? ((uint32_t)i * g.group + t) * 8 + j : ((uint32_t)(i * 8 + j)) * g.group + t; };

    float h[kN][8], z[kN][8];
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        if (kWide) {
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] = 0.0f;
            if (at(i, 0) < D) load8(x + at(i, 0), h[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] = at(i, j) < D ? load1(x + at(i, j)) : 0.0f;
        }
    }
    if (p.gate != nullptr) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            if (kWide) {
                if (at(i, 0) < D) load8(gate + at(i, 0), z[i]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) z[i][j] = at(i, j) < D ? load1(gate + at(i, j)) : 0.0f;
            }
        }
    }
    if (p.residual != nullptr) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            if (kWide) {
                if (at(i, 0) < D) {
                    float v[8];
                    load8(p.residual, res + at(i, 0), p.residual_type, v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[i][j] += v[j];
                    store8(p.residual, res + at(i, 0), p.residual_type, h[i]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (at(i, j) < D) {
                        h[i][j] += load1(p.residual, res + at(i, j), p.residual_type);
                        store1(p.residual, res + at(i, j), p.residual_type, h[i][j]);
                    }
            }
        }
    }
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kN; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(h[i][j], h[i][j], sum);
    sum = meet<false>(sum, g.group, false, partial[0]);
    const float f = rsqrtf(sum / (float)p.dim + p.eps);

    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        float w[8];
        if (p.weight != nullptr) {
            if (kWide) {
                if (at(i, 0) < D) load8(p.weight, at(i, 0), p.weight_type, w);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = at(i, j) < D ? load1(p.weight, at(i, j), p.weight_type) : 0.0f;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float y = h[i][j] * f;
            if (p.weight != nullptr) y *= w[j];
            if (p.gate != nullptr) y *= silu(z[i][j]);
            h[i][j] = y;
            if (at(i, kWide ? 0 : j) < D) top = larger(top, fabsf(y));
        }
    }
    const int64_t out = token * p.out_token + head * p.out_head;
    if (p.out_type == kE4M3) {
        top = meet<true>(top, g.group, g.token != 0, partial[1]);
        float scale = top / 448.0f;
        if (scale < 0x1p-126f) scale = 0x1p-126f; /* not for a NaN */
        const float inv = 1.0f / scale;
        if (live && t == 0 && head == 0) p.scales[token] = scale;
        uint8_t *o = static_cast<uint8_t *>(p.out) + out;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            if (kWide) {
                if (at(i, 0) < D) {
                    uint32_t w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        w[j] = __nv_cvt_float2_to_fp8x2(make_float2(h[i][2 * j] * inv, h[i][2 * j + 1] * inv), __NV_SATFINITE, __NV_E4M3);
                    *reinterpret_cast<uint2 *>(o + at(i, 0)) = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (at(i, j) < D) o[at(i, j)] = __nv_cvt_float_to_fp8(h[i][j] * inv, __NV_SATFINITE, __NV_E4M3);
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        if (kWide) {
            if (at(i, 0) < D) store8(p.out, out + at(i, 0), p.out_type, h[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (at(i, j) < D) store1(p.out, out + at(i, j), p.out_type, h[i][j]);
        }
    }
}

template <typename T, bool kWide, int kN>
cudaError_t launch_norm_t(const NormParams &p, cudaStream_t stream) {
    NormShape g;
    g.group = norm_group(p.dim, 8 * kN);
    g.token = p.out_type == kE4M3 && p.heads > 1;
    g.rows = g.token ? p.heads : g.group >= 128 ? 1 : 128 / g.group;
    const uint32_t block = (g.group * g.rows + 31) / 32 * 32;
    const uint64_t rows = (uint64_t)p.tokens * p.heads, grid = (rows + g.rows - 1) / g.rows;
    return launch(norm_kernel<T, kWide, kN>, dim3((uint32_t)grid), block, 0, stream, p, g);
}

/* rows of an operand that all start on a 16-byte boundary (8 bytes of 8-bit values) */
bool wide_rows(const void *p, int64_t token, int64_t head, const NormParams &n, int64_t size) {
    if (p == nullptr) return true;
    const int64_t step = 8 * size < 16 ? 8 : 16;
    return reinterpret_cast<uintptr_t>(p) % step == 0 && (n.tokens == 1 || token * size % step == 0) &&
           (n.heads == 1 || head * size % step == 0);
}

template <typename T>
cudaError_t launch_norm_x(const NormParams &p, cudaStream_t stream) {
    auto size = [](int type) { return type == kF32 ? 4 : type == kBF16 ? 2 : 1; };
    const bool wide = p.dim % 8 == 0 && wide_rows(p.x, p.x_token, p.x_head, p, sizeof(T)) &&
                      wide_rows(p.gate, p.gate_token, p.gate_head, p, sizeof(T)) &&
                      wide_rows(p.residual, p.residual_token, p.residual_head, p, size(p.residual_type)) &&
                      wide_rows(p.out, p.out_token, p.out_head, p, size(p.out_type)) && on16(p.weight);
    /* eight values a thread, or sixteen where a CTA would have too few threads */
    const bool two = norm_threads(p, 8) > kMaxNormThreads;
    auto *launch = wide ? two ? launch_norm_t<T, true, 2> : launch_norm_t<T, true, 1>
                        : two ? launch_norm_t<T, false, 2> : launch_norm_t<T, false, 1>;
    return launch(p, stream);
}

}  // namespace

cudaError_t launch_norm(const NormParams &p, int, cudaStream_t stream) {
    return p.type == kBF16 ? launch_norm_x<__nv_bfloat16>(p, stream) : launch_norm_x<float>(p, stream);
}

}  // namespace ops
}  // namespace gdn
