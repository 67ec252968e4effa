/* gdn_delta.cu -- the gated delta rule token by token over pooled states: the
 * new token of every decode stream, or a few tokens of each.
 *
 * Per value head, S [V][K] in FP32:
 *   r = S k,  p = S q                        (one pass over the old state)
 *   delta = beta (v - e^g r)
 *   o = scale (e^g p + (q.k) delta)          (= scale S' q)
 *   S' = e^g S + delta k^T
 * q and k are first divided by sqrt(sum x^2 + 1e-6) where asked for.
 *
 * Bound by the state's crossing of HBM once each way (V K 8 bytes a head
 * against 6 V K flops). A row of S is held by eight lanes, K / 8 values each
 * in registers: a warp's load takes whole 128-byte lines of four rows and a
 * row's two sums need three shuffles. The state is requested before the
 * token's vectors, so that their norms are formed while it arrives. q, k and
 * the scalars of up to a warp count of tokens are staged in shared memory in
 * FP32; the state stays in registers over all tokens of the sequence.
 */
#include "gdn_ops.h"

#include <cuda_bf16.h>

namespace gdn {
namespace ops {

namespace {

constexpr int kLanesPerRow = 8;
constexpr int kStepThreads = 256;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void store_out(float *p, float x) { *p = x; }
__device__ __forceinline__ void store_out(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

template <int K, typename T>
__global__ void __launch_bounds__(kStepThreads) delta_step_kernel(const __grid_constant__ DeltaParams p) {
    constexpr int kVec = K / kLanesPerRow / 4;   /* float4 of a row in a lane */
    constexpr int kMaxTile = kStepThreads / 32;  /* tokens staged at once: one per warp */
    __shared__ __align__(16) float qs[kMaxTile][K], ks[kMaxTile][K];
    __shared__ float vs[kMaxTile][32];
    __shared__ float dec[kMaxTile], bet[kMaxTile], alp[kMaxTile];
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nwarps = blockDim.x >> 5;
    const uint32_t rows = blockDim.x / kLanesPerRow, blocks = p.V / rows;
    const T *q = static_cast<const T *>(p.q), *k = static_cast<const T *>(p.k), *v = static_cast<const T *>(p.v);
    T *out = static_cast<T *>(p.out);

    const uint32_t n = blockIdx.x / (p.HV * blocks), rem = blockIdx.x - n * (p.HV * blocks);
    if (n == p.N) {
        /* tokens that no sequence covers (the last head's CTAs) give zeros */
        uint32_t first, t0, t1, last;
        sequence_tokens(p, 0, first, t0);
        sequence_tokens(p, p.N - 1, t1, last);
        const uint32_t width = p.HV * p.V;
        for (uint32_t t = 0; t < p.tokens; ++t) {
            if (t == first) t = last;
            if (t >= p.tokens) break;
            for (uint32_t i = rem * blockDim.x + tid; i < width; i += p.HV * blocks * blockDim.x)
                store_out(out + (int64_t)t * p.out_token + (int64_t)(i / p.V) * p.out_head + i % p.V, 0.0f);
        }
        return;
    }
    const uint32_t h = rem / blocks, row0 = (rem - h * blocks) * rows;
    const uint32_t hq = h / (p.HV / p.H);
    const uint32_t row = row0 + tid / kLanesPerRow, l8 = tid & (kLanesPerRow - 1);
    uint32_t t0, t1;
    sequence_tokens(p, n, t0, t1);
    const int64_t slot = sequence_slot(p, n);
    if (slot < 0) {
        for (uint32_t t = t0; t < t1; ++t)
            if (tid < rows) store_out(out + (int64_t)t * p.out_token + (int64_t)h * p.out_head + row0 + tid, 0.0f);
        return;
    }
    const bool fresh = p.fresh != nullptr && p.fresh[n] != 0;
    if (t0 == t1 && !fresh) return;

    float4 *S = reinterpret_cast<float4 *>(p.state + slot * p.state_slot + ((int64_t)h * p.V + row) * K) + l8;
    float4 s[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) s[j] = fresh ? make_float4(0.f, 0.f, 0.f, 0.f) : S[j * kLanesPerRow];

    for (uint32_t tile = t0; tile < t1; tile += nwarps) {
        if (tile != t0) __syncthreads();
        if (tile + warp < t1) {
            const int64_t t = tile + warp;
            const T *qt = q + t * p.q_token + (int64_t)hq * p.q_head, *kt = k + t * p.k_token + (int64_t)hq * p.k_head;
            float qv[K / 32], kv[K / 32], qq = 0.f, kk = 0.f, qk = 0.f;
#pragma unroll
            for (int i = 0; i < K / 32; ++i) {
                qv[i] = to_float(qt[lane + 32 * i]);
                kv[i] = to_float(kt[lane + 32 * i]);
            }
            const float vv = lane < rows ? to_float(v[t * p.v_token + (int64_t)h * p.v_head + row0 + lane]) : 0.f;
            const float gv = p.g[t * p.g_token + (int64_t)h * p.g_head];
            const float bv = p.beta[t * p.beta_token + (int64_t)h * p.beta_head];
#pragma unroll
            for (int i = 0; i < K / 32; ++i) {
                qq = fmaf(qv[i], qv[i], qq);
                kk = fmaf(kv[i], kv[i], kk);
                qk = fmaf(qv[i], kv[i], qk);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                qq += __shfl_xor_sync(0xffffffffu, qq, o);
                kk += __shfl_xor_sync(0xffffffffu, kk, o);
                qk += __shfl_xor_sync(0xffffffffu, qk, o);
            }
            const float qi = p.normalize ? p.scale / sqrtf(qq + 1e-6f) : p.scale;
            const float ki = p.normalize ? 1.0f / sqrtf(kk + 1e-6f) : 1.0f;
#pragma unroll
            for (int i = 0; i < K / 32; ++i) {
                qs[warp][lane + 32 * i] = qv[i] * qi;
                ks[warp][lane + 32 * i] = kv[i] * ki;
            }
            vs[warp][lane] = vv;
            if (lane == 0) {
                dec[warp] = expf(gv);
                bet[warp] = bv;
                alp[warp] = qk * qi * ki;
            }
        }
        __syncthreads();
        const uint32_t nt = min(nwarps, t1 - tile);
        for (uint32_t i = 0; i < nt; ++i) {
            const float4 *k4 = reinterpret_cast<const float4 *>(ks[i]) + l8;
            const float4 *q4 = reinterpret_cast<const float4 *>(qs[i]) + l8;
            float r0 = 0.f, r1 = 0.f, p0 = 0.f, p1 = 0.f;
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const float4 a = k4[j * kLanesPerRow], b = q4[j * kLanesPerRow];
                r0 = fmaf(s[j].x, a.x, r0);
                r1 = fmaf(s[j].y, a.y, r1);
                r0 = fmaf(s[j].z, a.z, r0);
                r1 = fmaf(s[j].w, a.w, r1);
                p0 = fmaf(s[j].x, b.x, p0);
                p1 = fmaf(s[j].y, b.y, p1);
                p0 = fmaf(s[j].z, b.z, p0);
                p1 = fmaf(s[j].w, b.w, p1);
            }
            float r = r0 + r1, pq = p0 + p1;
#pragma unroll
            for (int o = 1; o < kLanesPerRow; o <<= 1) {
                r += __shfl_xor_sync(0xffffffffu, r, o);
                pq += __shfl_xor_sync(0xffffffffu, pq, o);
            }
            const float d = dec[i];
            const float delta = bet[i] * (vs[i][tid / kLanesPerRow] - d * r);
            if (l8 == 0)
                store_out(out + (int64_t)(tile + i) * p.out_token + (int64_t)h * p.out_head + row,
                          d * pq + alp[i] * delta);
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const float4 a = k4[j * kLanesPerRow];
                s[j].x = fmaf(d, s[j].x, a.x * delta);
                s[j].y = fmaf(d, s[j].y, a.y * delta);
                s[j].z = fmaf(d, s[j].z, a.z * delta);
                s[j].w = fmaf(d, s[j].w, a.w * delta);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < kVec; ++j) S[j * kLanesPerRow] = s[j];
}

template <int K>
cudaError_t launch_step_k(const DeltaParams &p, bool bf16, cudaStream_t stream) {
    const uint32_t rows = kStepThreads / kLanesPerRow;
    const uint32_t grid = (p.N + (p.starts != nullptr ? 1u : 0u)) * p.HV * (p.V / rows);
    if (bf16)
        delta_step_kernel<K, __nv_bfloat16><<<grid, kStepThreads, 0, stream>>>(p);
    else
        delta_step_kernel<K, float><<<grid, kStepThreads, 0, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_delta_step(const DeltaParams &p, bool bf16, cudaStream_t stream) {
    switch (p.K) {
        case 64: return launch_step_k<64>(p, bf16, stream);
        case 128: return launch_step_k<128>(p, bf16, stream);
        default: return launch_step_k<256>(p, bf16, stream);
    }
}

}  // namespace ops
}  // namespace gdn
