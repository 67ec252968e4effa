/* gdn_linear_few.cu -- y = act(sx sw x W^T + bias) + residual for up to 16
 * tokens (gdn_linear.cu takes more, and 9 and more with many weights).
 *
 * Bound by reading W once. A warp multiplies 16 rows of W with 8 (or 16)
 * tokens by m16n8k16 MMAs whose operands come straight from memory: in a
 * fragment, lane (g, t) = (lane / 4, lane % 4) holds values of row g of W and of token
 * g at four places of k. Which k stand there is free as long as both operands
 * agree, so each lane loads 16 bytes, neighbours in k, of rows g and g + 8 and
 * of token g, and feeds them to two MMAs (8-bit values, exact in FP16, to
 * four). Nothing passes through shared memory but the sums: the warps of a CTA
 * share its rows and divide k between them, and their partial sums are added in
 * the order of the warps.
 *
 * Measured: one token of 2048 inputs by 8208 outputs of BF16 6.9 us (4.9 TB/s),
 * by 32000 19.1 us (6.9 TB/s, the rate of a copy), of 8 bits 6.2 and 14.5 us;
 * what small calls take above the bytes is the launch and one wait for memory,
 * about 2.5 us, and in 8 bits the conversions to FP16: four of W and two of each eight tokens an MMA. 16 tokens
 * read as much of x as of W: 12.1 and 29.4 us. With swiglu they spill 88 (BF16) and 120 bytes a thread (2048 by 2 x 2048
 * 6.2 us).
 */
#include "gdn_linear.h"

namespace gdn {
namespace ops {

namespace {

constexpr uint32_t kMaxWarps = 16;

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
/* two values of 8 bits as two of 16 */
__device__ __forceinline__ uint32_t widen(uint32_t two) {
    uint32_t r;
    asm("{\n .reg .b16 h;\n cvt.u16.u32 h, %1;\n cvt.rn.f16x2.e4m3x2 %0, h;\n}\n" : "=r"(r) : "r"(two));
    return r;
}

/* 16 bytes of row g, of row g + 8 and of a token: their products */
template <bool kFp8, int kGroups>
__device__ __forceinline__ void products(float (&d)[kGroups][4], const uint4 &lo, const uint4 &hi, const uint4 (&b)[kGroups]) {
    const uint32_t l[4] = {lo.x, lo.y, lo.z, lo.w}, h[4] = {hi.x, hi.y, hi.z, hi.w};
    if constexpr (kFp8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t a0 = widen(l[i] & 0xFFFFu), a1 = widen(h[i] & 0xFFFFu), a2 = widen(l[i] >> 16), a3 = widen(h[i] >> 16);
#pragma unroll
            for (int n = 0; n < kGroups; ++n) {
                const uint32_t w = i == 0 ? b[n].x : i == 1 ? b[n].y : i == 2 ? b[n].z : b[n].w;
                mma_f16(d[n], a0, a1, a2, a3, widen(w & 0xFFFFu), widen(w >> 16));
            }
        }
    } else {
#pragma unroll
        for (int n = 0; n < kGroups; ++n) {
            mma_bf16(d[n], l[0], h[0], l[1], h[1], b[n].x, b[n].y);
            mma_bf16(d[n], l[2], h[2], l[3], h[3], b[n].z, b[n].w);
        }
    }
}

/* weights: read once */
__device__ __forceinline__ uint4 load16(const uint8_t *p) {
    uint4 v;
    asm volatile("ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
/* 16 bytes at byte k of a row of `size` bytes, zeros past its end */
template <bool kFp8>
__device__ __forceinline__ uint4 piece(const uint8_t *row, uint32_t k, uint32_t size) {
    if (k >= size) return make_uint4(0, 0, 0, 0);
    if (k + 16 <= size) return __ldcg(reinterpret_cast<const uint4 *>(row + k));
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; i += kFp8 ? 1 : 2)
        if (k + i < size) {
            const uint32_t e = kFp8 ? (uint32_t)__ldcg(row + k + i) : (uint32_t)__ldcg(reinterpret_cast<const unsigned short *>(row + k + i));
            w[i / 4] |= e << (8 * (i % 4));
        }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

/* Steps of k (64 bytes of a row) at a time, while the next ones' loads are in flight: what 128 registers hold. */
__host__ __device__ constexpr int ahead_of(int products) { return products == 1 ? 4 : 2; }

/* kGroups: tokens / 8. kPairs (swiglu): a CTA takes 16 rows of either half of W. */
template <bool kFp8, int kGroups, bool kPairs>
__global__ void __launch_bounds__(kMaxWarps * 32) linear_few_kernel(const __grid_constant__ LinearParams p) {
    constexpr int kHalves = kPairs ? 2 : 1;
    constexpr int kAhead = ahead_of(kGroups * kHalves);
    constexpr uint32_t kSums = kHalves * kGroups * 128; /* of a warp */
    extern __shared__ float sums[];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, warps = blockDim.x >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const uint32_t n0 = blockIdx.x * 16, size = p.inputs * (kFp8 ? 1 : 2);
    const uint32_t elem = kFp8 ? 1 : 2;
    /* rows past the ends are read as the last one: their sums go nowhere */
    const uint8_t *w[kHalves][2], *x[kGroups];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
            w[h][r] = static_cast<const uint8_t *>(p.weight) + (h * p.outputs + min(n0 + g + 8 * r, p.outputs - 1)) * p.weight_row * elem + t * 16;
#pragma unroll
    for (int n = 0; n < kGroups; ++n) x[n] = static_cast<const uint8_t *>(p.x) + min(g + 8 * n, p.tokens - 1) * p.x_row * elem + t * 16;
    float d[kHalves][kGroups][4];
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int n = 0; n < kGroups; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) d[h][n][i] = 0.0f;

    const uint32_t whole = size / (kAhead * 64) * (kAhead * 64), stride = warps * kAhead * 64;
    uint32_t k0 = warp * kAhead * 64;
    /* Before the kernel before this one has ended, the first rows of W are on their way to L2 (which the loads below
     * read: they see what that kernel wrote). One row of 2048 by 8208 of BF16 7.1 us instead of 8.1, by 2048 3.1 instead
     * of 3.5; all of a warp's rows 7.9. 8-bit rows without pairs do not gain (by 32000 15.4 us instead of 14.9). */
    if ((!kFp8 || kPairs) && k0 < whole) {
#pragma unroll
        for (int s = 0; s < kAhead; ++s)
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
#pragma unroll
                for (int r = 0; r < 2; ++r) asm volatile("prefetch.global.L2 [%0];" ::"l"(w[h][r] + k0 + s * 64));
    }
    wait_for_previous();
    let_next_start();
    struct Loads {
        uint4 a[kAhead][kHalves][2], b[kAhead][kGroups];
    };
    auto load = [&](Loads &l, uint32_t k0) {
#pragma unroll
        for (int s = 0; s < kAhead; ++s) {
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
#pragma unroll
                for (int r = 0; r < 2; ++r) l.a[s][h][r] = load16(w[h][r] + k0 + s * 64);
#pragma unroll
            for (int n = 0; n < kGroups; ++n) l.b[s][n] = __ldcg(reinterpret_cast<const uint4 *>(x[n] + k0 + s * 64));
        }
    };
    /* The tensor cores cut their sums towards zero: the ones of a set are added to the others with rounding to nearest. In
     * one sum of 1408 inputs a warp, results of 5632 inputs were 1.4e-6 off in the 2-norm, 2.9e-6 of swiglu; so 1.4e-7
     * and 2.0e-7, at no cost but for 16 tokens of swiglu (2048 by 2 x 5632 15.2 us instead of 14.4, for want of registers). */
    auto multiply = [&](const Loads &l) {
        float part[kHalves][kGroups][4] = {};
#pragma unroll
        for (int s = 0; s < kAhead; ++s)
#pragma unroll
            for (int h = 0; h < kHalves; ++h) products<kFp8, kGroups>(part[h], l.a[s][h][0], l.a[s][h][1], l.b[s]);
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
#pragma unroll
            for (int n = 0; n < kGroups; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) d[h][n][i] += part[h][n][i];
    };
    /* the whole steps, in turn over the warps, each time with the next one's loads under way */
    Loads one, two;
    if (k0 < whole) load(one, k0);
    while (k0 < whole) {
        if (k0 + stride < whole) load(two, k0 + stride);
        multiply(one);
        k0 += stride;
        if (k0 >= whole) break;
        if (k0 + stride < whole) load(one, k0 + stride);
        multiply(two);
        k0 += stride;
    }
    /* the rest of a row */
    for (uint32_t k = whole + warp * 64; k < size; k += warps * 64) {
        uint4 b[kGroups];
#pragma unroll
        for (int n = 0; n < kGroups; ++n) b[n] = piece<kFp8>(x[n] - t * 16, k + t * 16, size);
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
            products<kFp8, kGroups>(d[h], piece<kFp8>(w[h][0] - t * 16, k + t * 16, size), piece<kFp8>(w[h][1] - t * 16, k + t * 16, size), b);
    }
    /* the warps' sums: [warp][half][token][16 rows] */
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int n = 0; n < kGroups; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                sums[warp * kSums + (h * kGroups * 8 + n * 8 + t * 2 + (i & 1)) * 16 + g + 8 * (i >> 1)] = d[h][n][i];
    __syncthreads();
    for (uint32_t i = tid; i < kGroups * 128; i += blockDim.x) {
        const uint32_t token = i / 16, n = n0 + i % 16;
        if (token >= p.tokens || n >= p.outputs) continue;
        float v[2] = {0.0f, 0.0f};
        for (uint32_t q = 0; q < warps; ++q)
#pragma unroll
            for (int h = 0; h < kHalves; ++h) v[h] += sums[q * kSums + h * kGroups * 128 + i];
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            const uint32_t row = h * p.outputs + n;
            if (kFp8) v[h] *= __ldcg(p.x_scales + token) * __ldcg(p.weight_scales + row);
            if (p.bias != nullptr) v[h] += load1(p.bias, row, p.bias_type);
        }
        float y = activate(p.activation, v[0], v[1]);
        if (p.residual != nullptr) y += load1(p.residual, token * p.residual_row + n, p.residual_type);
        store1(p.out, token * p.out_row + n, p.out_type, y);
    }
}

template <bool kFp8, int kGroups, bool kPairs>
cudaError_t launch_few_t(const LinearParams &p, int sms, cudaStream_t stream) {
    const uint32_t ctas = (p.outputs + 15) / 16;
    constexpr int kAhead = ahead_of(kGroups * (kPairs ? 2 : 1));
    /* as many warps as let all CTAs run at once (about 20 an SM), as far as k goes round */
    const uint32_t steps = (p.inputs * (kFp8 ? 1 : 2) + kAhead * 64 - 1) / (kAhead * 64);
    uint32_t warps = ctas <= (uint32_t)sms ? kMaxWarps : ctas <= 2u * (uint32_t)sms ? 8 : 4;
    while (warps > 1 && warps > steps) warps /= 2;
    const size_t smem = (size_t)warps * (kPairs ? 2 : 1) * kGroups * 128 * sizeof(float);
    return launch_overlapped(linear_few_kernel<kFp8, kGroups, kPairs>, dim3(ctas), warps * 32, smem, stream, p);
}

template <bool kFp8>
cudaError_t launch_few_x(const LinearParams &p, int sms, cudaStream_t stream) {
    const bool two = p.tokens > 8;
    if (p.activation == kSwiglu)
        return two ? launch_few_t<kFp8, 2, true>(p, sms, stream) : launch_few_t<kFp8, 1, true>(p, sms, stream);
    return two ? launch_few_t<kFp8, 2, false>(p, sms, stream) : launch_few_t<kFp8, 1, false>(p, sms, stream);
}

}  // namespace

/* More than eight tokens double what this kernel reads of x, and it slows down where there are many weights; the other's
 * tiles take 5 us at least. 16 tokens of 2048 by 2048 4.2 us here and 6.7 there, of 5632 by 2048 7.4 and 9.6 (8 bits 5.9 and
 * 7.5), of 2048 by 8208 12.1 and 10.1 (8 bits 8.9 and 7.1), by 2 x 5632 15.2 and 12.9 (11.8 and 8.7), by 32000 29.4 and 26.8
 * (20.1 and 17.8); 8 tokens by 32000 23.0. */
bool takes_few(const LinearParams &p) {
    return p.tokens <= 8 || (p.tokens <= kFewTokens && (uint64_t)p.inputs * p.outputs * (p.activation == kSwiglu ? 2 : 1) <= 14000000u);
}

cudaError_t launch_linear_few(const LinearParams &p, int sms, cudaStream_t stream) {
    return p.type == kE4M3 ? launch_few_x<true>(p, sms, stream) : launch_few_x<false>(p, sms, stream);
}

}  // namespace ops
}  // namespace gdn
