/* gdn_logits.cu -- constraints on the logits of a set of streams, and the
 * greedy pick. For a row x [V], a token v that the row's history holds n
 * times after its prompt and m times in all:
 *   m > 0:  x = x > 0 ? x / r : x r          (repetition)
 *   n > 0:  x = (x - f n) - p                (frequency, presence)
 *   x = x + (sum of the row's biases of v, in list order)
 *   mask bit of v clear: x = -inf
 * rounded once to the logits' type; the pick is the lowest index of the
 * largest written value (NaN never, -1 if none is above -inf). Each operation
 * is one FP32 rounding, so results do not depend on the split.
 *
 * Bound by HBM: every logit is read and written once. A row is cut into the
 * slices of one cluster's CTAs. Each CTA reads the row's history and keeps
 * what falls into its slice in a shared-memory table, one word per token:
 *   bits 0-19 n | bits 20-30 first bias entry + 1 | bit 31 in the prompt
 * (integer atomics: the order does not show), and one bit per token that says
 * whether the word is set. Tokens without one (nearly all) only meet the mask:
 * a dense pass copies them 16 bytes at a time and keeps the largest. The few
 * others are then recomputed from the history and bias lists themselves: who
 * takes a token's word out of the table (an exchange with 0) does the token,
 * so that all lanes of a warp have one to do, where a test in the dense pass
 * left a warp waiting for one lane at nearly every vector. The picks of the
 * slices meet in CTA 0 through distributed shared memory.
 */
#include "gdn_ops.h"

#include <cooperative_groups.h>
#include <cuda_bf16.h>

namespace gdn {
namespace ops {

namespace {

namespace cg = cooperative_groups;

constexpr int kLogitsThreads = 512;
constexpr int kUnroll = 4;      /* 16-byte vectors of a thread in flight */
constexpr int kHistoryUnroll = 4;
constexpr int kMaxCluster = 8;  /* portable cluster size */
constexpr uint32_t kCountMask = (1u << 20) - 1, kPromptBit = 1u << 31;
constexpr uint32_t kFlagWords = (kMaxBiases + 32) / 32;

/* pick key: larger value first, then the lower index; NaN is 0 and so never wins */
__device__ __forceinline__ unsigned long long pick_key(float x, uint32_t v) {
    if (x != x) return 0ull;
    uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);
    b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return ((unsigned long long)b << 32) | (unsigned long long)(0xFFFFFFFFu - v);
}
constexpr uint32_t kKeyNegInf = 0x007FFFFFu; /* value half of the key of -inf */

/* 16 bytes of logits. only(allow): the values whose bit is set, -inf for the others. */
template <typename T>
struct Vec;
template <>
struct Vec<float> {
    static constexpr int kN = 4;
    static __device__ __forceinline__ float value(const uint4 &w, int j) {
        return __uint_as_float(j == 0 ? w.x : j == 1 ? w.y : j == 2 ? w.z : w.w);
    }
    static __device__ __forceinline__ uint4 only(const uint4 &w, uint32_t allow) {
        return make_uint4((allow & 1u) ? w.x : 0xFF800000u, (allow & 2u) ? w.y : 0xFF800000u,
                          (allow & 4u) ? w.z : 0xFF800000u, (allow & 8u) ? w.w : 0xFF800000u);
    }
    /* largest value, NaN passed over (-inf if there is nothing else) */
    static __device__ __forceinline__ float largest(const uint4 &w) {
        const float lo = __int_as_float(0xff800000);
        return fmaxf(fmaxf(fmaxf(__uint_as_float(w.x), lo), __uint_as_float(w.y)),
                     fmaxf(fmaxf(__uint_as_float(w.z), lo), __uint_as_float(w.w)));
    }
};
template <>
struct Vec<__nv_bfloat16> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ float value(const uint4 &w, int j) {
        const uint32_t u = j < 2 ? w.x : j < 4 ? w.y : j < 6 ? w.z : w.w;
        return __uint_as_float((j & 1) ? (u & 0xFFFF0000u) : (u << 16));
    }
    static __device__ __forceinline__ uint32_t pair(uint32_t w, uint32_t allow) {
        const uint32_t m = ((allow & 1u) | ((allow & 2u) << 15)) * 0xFFFFu;
        return (w & m) | (0xFF80FF80u & ~m);
    }
    static __device__ __forceinline__ uint4 only(const uint4 &w, uint32_t allow) {
        return make_uint4(pair(w.x, allow), pair(w.y, allow >> 2), pair(w.z, allow >> 4), pair(w.w, allow >> 6));
    }
    static __device__ __forceinline__ __nv_bfloat162 two(uint32_t w) { return *reinterpret_cast<__nv_bfloat162 *>(&w); }
    static __device__ __forceinline__ float largest(const uint4 &w) {
        const __nv_bfloat162 lo = two(0xFF80FF80u);
        const __nv_bfloat162 m = __hmax2(__hmax2(__hmax2(two(w.x), lo), two(w.y)), __hmax2(__hmax2(two(w.z), lo), two(w.w)));
        return fmaxf(__low2float(m), __high2float(m));
    }
};
__device__ __forceinline__ float load_one(const float *p) { return *p; }
__device__ __forceinline__ float load_one(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ float rounded(float x, float) { return x; }
__device__ __forceinline__ float rounded(float x, __nv_bfloat16) { return __bfloat162float(__float2bfloat16_rn(x)); }
__device__ __forceinline__ void store_one(float *p, float x) { *p = x; }
__device__ __forceinline__ void store_one(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

struct Row {
    float repetition, presence, frequency;
    const int32_t *bias_ids;
    const float *bias;
    const uint32_t *multi; /* bias entries whose token has later entries too */
    uint32_t biases;
};

/* x with what the table's word says */
__device__ __forceinline__ float touched(float x, uint32_t word, const Row &r) {
    const uint32_t n = word & kCountMask, entry = (word >> 20) & kMaxBiases;
    if (n != 0 || (word & kPromptBit)) x = x > 0.0f ? __fdiv_rn(x, r.repetition) : __fmul_rn(x, r.repetition);
    if (n != 0) x = __fsub_rn(__fsub_rn(x, __fmul_rn(r.frequency, (float)n)), r.presence);
    if (entry != 0) {
        const uint32_t i = entry - 1;
        float sum = r.bias[i];
        if ((r.multi[i >> 5] >> (i & 31)) & 1u)
            for (uint32_t j = i + 1; j < r.biases; ++j)
                if (r.bias_ids[j] == r.bias_ids[i]) sum = __fadd_rn(sum, r.bias[j]);
        x = __fadd_rn(x, sum);
    }
    return x;
}

template <typename T>
__global__ void __launch_bounds__(kLogitsThreads) logits_kernel(const __grid_constant__ LogitsParams p) {
    constexpr int N = Vec<T>::kN;
    extern __shared__ __align__(16) uint32_t table[]; /* words of the slice, then a bit each */
    __shared__ uint32_t multi[kFlagWords];
    __shared__ unsigned long long warp_key[kLogitsThreads / 32], slice_key[kMaxCluster];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t C = cluster.num_blocks(), rank = cluster.block_rank(), b = blockIdx.x / C;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T *in = static_cast<const T *>(p.logits) + (int64_t)b * p.logits_row;
    T *out = static_cast<T *>(p.out) + (int64_t)b * p.out_row;
    const uint32_t V = p.vocab;
    /* vectors are cut at 16-byte boundaries of the input row: vector i holds
     * the tokens i N - mis .. i N - mis + N - 1 */
    const uint32_t mis = (uint32_t)((reinterpret_cast<uintptr_t>(in) / sizeof(T)) % N);
    const bool wide_out = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    const uint32_t nvec = (mis + V + N - 1) / N;
    const uint32_t v0 = min(nvec, rank * p.slice_vecs), v1 = min(nvec, v0 + p.slice_vecs);
    const int32_t first = (int32_t)(v0 * N) - (int32_t)mis; /* token of table word 0 */
    const int32_t lo = max(first, 0), hi = min((int32_t)V, (int32_t)(v1 * N) - (int32_t)mis);
    const uint32_t *mask = p.mask == nullptr ? nullptr : p.mask + (int64_t)b * p.mask_row;
    const uint32_t words = (p.slice_vecs * N + 127) & ~127u;
    uint32_t *bits = table + words;

    uint4 w[kUnroll];
    /* the vectors base, base + kLogitsThreads, ... that lie in the row whole */
    auto whole = [&](uint32_t i) {
        const int32_t e0 = (int32_t)(i * N) - (int32_t)mis;
        return i < v1 && e0 >= 0 && e0 + N <= (int32_t)V;
    };
    auto load = [&](uint32_t base) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const uint32_t i = base + u * kLogitsThreads;
            if (whole(i)) w[u] = __ldcs(reinterpret_cast<const uint4 *>(in + ((int32_t)(i * N) - (int32_t)mis)));
        }
    };
    load(v0 + tid); /* on their way while the table is built */

    const bool use_table = p.tokens != nullptr || p.bias_ids != nullptr;
    Row row;
    row.repetition = p.repetition == nullptr ? 1.0f : p.repetition[b];
    row.presence = p.presence == nullptr ? 0.0f : p.presence[b];
    row.frequency = p.frequency == nullptr ? 0.0f : p.frequency[b];
    row.bias_ids = p.bias_ids + (int64_t)b * p.bias_ids_row;
    row.bias = p.bias + (int64_t)b * p.bias_row;
    row.multi = multi;
    row.biases = p.bias_ids == nullptr ? 0 : p.biases;
    const int32_t *ids = p.tokens + (int64_t)b * p.tokens_row;
    const int32_t len = p.tokens == nullptr ? 0 : p.lens == nullptr ? (int32_t)p.history : min(p.lens[b], (int32_t)p.history);

    if (use_table) {
        for (uint32_t i = tid; i < (words + words / 32) / 4; i += kLogitsThreads)
            reinterpret_cast<uint4 *>(table)[i] = make_uint4(0, 0, 0, 0);
        for (uint32_t i = tid; i < kFlagWords; i += kLogitsThreads) multi[i] = 0;
        __syncthreads();
        const int32_t made = p.prompt_lens == nullptr ? 0 : p.prompt_lens[b];
        for (int32_t i0 = (int32_t)tid; i0 < len; i0 += kLogitsThreads * kHistoryUnroll) {
            int32_t id[kHistoryUnroll];
#pragma unroll
            for (int u = 0; u < kHistoryUnroll; ++u) {
                const int32_t i = i0 + u * kLogitsThreads;
                id[u] = i < len ? ids[i] : -1;
            }
#pragma unroll
            for (int u = 0; u < kHistoryUnroll; ++u) {
                if (id[u] < lo || id[u] >= hi) continue;
                const uint32_t at = (uint32_t)(id[u] - first);
                const uint32_t old = i0 + u * kLogitsThreads >= made ? atomicAdd(&table[at], 1u) : atomicOr(&table[at], kPromptBit);
                if (old == 0) atomicOr(&bits[at >> 5], 1u << (at & 31));
            }
        }
        /* a biased token's word names its first entry */
        for (uint32_t i = tid; i < row.biases; i += kLogitsThreads) {
            const int32_t id = row.bias_ids[i];
            if (id < lo || id >= hi) continue;
            const uint32_t at = (uint32_t)(id - first);
            uint32_t old = table[at];
            while (true) {
                const uint32_t e = (old >> 20) & kMaxBiases;
                if (e != 0 && e <= i + 1) break;
                const uint32_t seen = atomicCAS(&table[at], old, (old & ~(kMaxBiases << 20)) | ((i + 1) << 20));
                if (seen == old) break;
                old = seen;
            }
            atomicOr(&bits[at >> 5], 1u << (at & 31));
        }
        __syncthreads();
        for (uint32_t i = tid; i < row.biases; i += kLogitsThreads) {
            const int32_t id = row.bias_ids[i];
            if (id < lo || id >= hi) continue;
            const uint32_t e = (table[id - first] >> 20) & kMaxBiases;
            if (e != i + 1) atomicOr(&multi[(e - 1) >> 5], 1u << ((e - 1) & 31));
        }
    }

    /* dense pass: the mask, and the largest of the tokens without a word.
     * Tokens with one keep their value for now. */
    unsigned long long best = 0;
    float top = __int_as_float(0xff800000);
    uint32_t top_vec = 0;
    uint4 top_w = make_uint4(0, 0, 0, 0);
    for (uint32_t base = v0 + tid; base < v1; base += kLogitsThreads * kUnroll) {
        if (base != v0 + tid) load(base);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const uint32_t i = base + u * kLogitsThreads;
            if (i >= v1) continue;
            const int32_t e0 = (int32_t)(i * N) - (int32_t)mis;
            const uint32_t at = (i - v0) * N;
            const uint32_t own = use_table ? bits[at >> 5] >> (at & 31) : 0u;
            if (!whole(i)) {
                /* a row's ragged first or last vector */
                for (int32_t e = max(e0, 0); e < min(e0 + N, (int32_t)V); ++e) {
                    float x = load_one(in + e);
                    if ((own >> (e - e0)) & 1u) {
                        store_one(out + e, x);
                        continue;
                    }
                    if (mask != nullptr && !((mask[e >> 5] >> (e & 31)) & 1u)) x = __int_as_float(0xff800000);
                    store_one(out + e, x);
                    const unsigned long long key = pick_key(x, (uint32_t)e);
                    best = key > best ? key : best;
                }
                continue;
            }
            uint32_t allow = 0xFFFFFFFFu;
            if (mask != nullptr) allow = __funnelshift_r(mask[e0 >> 5], mask[(e0 + N - 1) >> 5], e0 & 31);
            const uint4 o = Vec<T>::only(w[u], allow | own);
            if (wide_out) {
                __stcs(reinterpret_cast<uint4 *>(out + e0), o);
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) store_one(out + e0 + j, Vec<T>::value(o, j));
            }
            const uint4 free = (own & ((1u << N) - 1)) ? Vec<T>::only(w[u], allow & ~own) : o;
            const float m = Vec<T>::largest(free);
            if (m > top) {
                top = m;
                top_vec = i;
                top_w = free;
            }
        }
    }
    if (top > __int_as_float(0xff800000)) {
#pragma unroll
        for (int j = N - 1; j >= 0; --j)
            if (Vec<T>::value(top_w, j) == top) {
                const unsigned long long key = pick_key(top, top_vec * N - mis + j);
                best = key > best ? key : best;
            }
    }
    if (use_table) {
        __syncthreads();
        auto recompute = [&](int32_t id) {
            if (id < lo || id >= hi) return;
            const uint32_t word = atomicExch(&table[id - first], 0u);
            if (word == 0) return;
            /* from out where the dense pass left it: out may be the logits */
            float x = touched(load_one(out + id), word, row);
            if (mask != nullptr && !((mask[id >> 5] >> (id & 31)) & 1u)) x = __int_as_float(0xff800000);
            x = rounded(x, T());
            store_one(out + id, x);
            const unsigned long long key = pick_key(x, (uint32_t)id);
            best = key > best ? key : best;
        };
        for (int32_t i0 = (int32_t)tid; i0 < len; i0 += kLogitsThreads * kHistoryUnroll) {
            int32_t id[kHistoryUnroll];
#pragma unroll
            for (int u = 0; u < kHistoryUnroll; ++u) {
                const int32_t i = i0 + u * kLogitsThreads;
                id[u] = i < len ? ids[i] : -1;
            }
#pragma unroll
            for (int u = 0; u < kHistoryUnroll; ++u) recompute(id[u]);
        }
        for (uint32_t i = tid; i < row.biases; i += kLogitsThreads) recompute(row.bias_ids[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
    }
    if (lane == 0) warp_key[warp] = best;
    __syncthreads();
    if (warp == 0) {
        best = lane < kLogitsThreads / 32 ? warp_key[lane] : 0ull;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
            best = other > best ? other : best;
        }
        if (lane == 0) cluster.map_shared_rank(slice_key, 0)[rank] = best;
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
        for (uint32_t c = 0; c < C; ++c) best = slice_key[c] > best ? slice_key[c] : best;
        p.picks[b] = (uint32_t)(best >> 32) > kKeyNegInf ? (int32_t)(0xFFFFFFFFu - (uint32_t)best) : -1;
    }
}

template <typename T>
cudaError_t launch_logits_t(LogitsParams &p, int sms, cudaStream_t stream) {
    constexpr uint32_t N = Vec<T>::kN;
    const uint32_t nvec = (p.vocab + N - 1) / N + 1; /* a row that starts inside a vector has one more */
    uint32_t C = 1;
    while (C < kMaxCluster && (p.rows * C < 2u * (uint32_t)sms || nvec * N / C > 16384u)) C *= 2;
    p.slice_vecs = (nvec + C - 1) / C;
    const bool use_table = p.tokens != nullptr || p.bias_ids != nullptr;
    const size_t words = (p.slice_vecs * N + 127) & ~127u;
    const size_t smem = use_table ? (words + words / 32) * 4 : 0;
    cudaError_t e = cudaFuncSetAttribute(logits_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.rows * C);
    cfg.blockDim = dim3(kLogitsThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, logits_kernel<T>, p);
}

}  // namespace

cudaError_t launch_logits(LogitsParams p, bool bf16, int sms, cudaStream_t stream) {
    return bf16 ? launch_logits_t<__nv_bfloat16>(p, sms, stream) : launch_logits_t<float>(p, sms, stream);
}

}  // namespace ops
}  // namespace gdn
