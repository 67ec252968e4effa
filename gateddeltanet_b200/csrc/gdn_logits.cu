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
 * slices of one cluster's CTAs. Each CTA reads the row's history and counts
 * what falls into its slice in shared memory (integer atomics: the order does
 * not show): n per token, in 16 bits where the logits have 16 and the history
 * is short enough, and a bit that history holds the token; another bit says
 * that a bias names it. The tokens with a bit, a few of a hundred, are found from
 * the bits and computed a lane each, and their results take the place of their
 * counts. The other tokens only meet the mask: a dense pass copies 16 bytes at
 * a time, puts in the results where a bit is set, and keeps the largest. (As
 * cases of the dense pass the few left whole warps waiting for the lanes that
 * had one: 135 us for 256 rows of 131072 BF16; computed after it, from what it
 * had written, they were a second round trip to memory: 71 us.) What bounds
 * the kernel beside HBM are the instructions that a warp spends once, so a CTA
 * has few warps with many logits each. The picks of the slices meet in CTA 0
 * through distributed shared memory.
 */
#include "gdn_ops.h"

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <type_traits>

namespace gdn {
namespace ops {

namespace {

namespace cg = cooperative_groups;

constexpr uint32_t kThreads = 256;
/* 16-byte vectors of a thread in flight: with four, four CTAs share an SM, with
 * two, five (256 rows of 131072 BF16 68 and 65 us, although 48 registers a thread
 * make it spill: 8 bytes in the aligned BF16 form, up to 28 in the others) */
constexpr int kUnroll = 2;
constexpr int kHistoryUnroll = 8;
constexpr int kMaxCluster = 8;  /* portable cluster size */

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
    /* w, with the values of t whose bit is set */
    static __device__ __forceinline__ uint4 blend(const uint4 &w, const uint4 &t, uint32_t own) {
        return make_uint4((own & 1u) ? t.x : w.x, (own & 2u) ? t.y : w.y, (own & 4u) ? t.z : w.z, (own & 8u) ? t.w : w.w);
    }
    static __device__ __forceinline__ uint32_t bits(float x) { return __float_as_uint(x); }
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
    /* of two values those of `yes` whose bit is set, those of `no` for the others */
    static __device__ __forceinline__ uint32_t pair(uint32_t yes, uint32_t no, uint32_t set) {
        const uint32_t m = ((set & 1u) | ((set & 2u) << 15)) * 0xFFFFu;
        return (yes & m) | (no & ~m);
    }
    static __device__ __forceinline__ uint4 blend(const uint4 &w, const uint4 &t, uint32_t own) {
        return make_uint4(pair(t.x, w.x, own), pair(t.y, w.y, own >> 2), pair(t.z, w.z, own >> 4), pair(t.w, w.w, own >> 6));
    }
    static __device__ __forceinline__ uint4 only(const uint4 &w, uint32_t allow) {
        constexpr uint32_t kNone = 0xFF80FF80u;
        return make_uint4(pair(w.x, kNone, allow), pair(w.y, kNone, allow >> 2), pair(w.z, kNone, allow >> 4),
                          pair(w.w, kNone, allow >> 6));
    }
    static __device__ __forceinline__ uint32_t bits(float x) { return __bfloat16_as_ushort(__float2bfloat16_rn(x)); }
    static __device__ __forceinline__ __nv_bfloat162 two(uint32_t w) { return *reinterpret_cast<__nv_bfloat162 *>(&w); }
    static __device__ __forceinline__ float largest(const uint4 &w) {
        const __nv_bfloat162 lo = two(0xFF80FF80u);
        const __nv_bfloat162 m = __hmax2(__hmax2(__hmax2(two(w.x), lo), two(w.y)), __hmax2(__hmax2(two(w.z), lo), two(w.w)));
        return fmaxf(__low2float(m), __high2float(m));
    }
};
__device__ __forceinline__ float load_one(const float *p) { return *p; }
__device__ __forceinline__ float load_one(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ float from_bits(uint32_t u, float) { return __uint_as_float(u); }
__device__ __forceinline__ float from_bits(uint32_t u, __nv_bfloat16) { return __uint_as_float(u << 16); }
__device__ __forceinline__ void store_one(float *p, float x) { *p = x; }
__device__ __forceinline__ void store_one(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

/* position of the n-th set bit (from 0) of a word that has more than n */
__device__ __forceinline__ uint32_t nth_bit(uint32_t w, uint32_t n) {
    uint32_t at = 0;
#pragma unroll
    for (uint32_t half = 16; half > 0; half >>= 1) {
        const uint32_t below = __popc(w & ((1u << half) - 1));
        if (n >= below) {
            n -= below;
            w >>= half;
            at += half;
        }
    }
    return at;
}

/* W: the type of a token's count, as wide as T or wider. kAligned: every row of logits and of out
 * starts on a 16-byte boundary. */
template <typename T, typename W, bool kAligned>
__global__ void __launch_bounds__(kThreads, 5) logits_kernel(const __grid_constant__ LogitsParams p) {
    constexpr int N = Vec<T>::kN;
    constexpr float kNegInf = -__builtin_huge_valf();
    extern __shared__ __align__(16) uint32_t table[]; /* counts of the slice, two bits each, the slice's biases */
    __shared__ unsigned long long warp_key[kThreads / 32], slice_key[kMaxCluster];
    __shared__ uint32_t slice_biases;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t C = cluster.num_blocks(), rank = cluster.block_rank(), b = blockIdx.x / C;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    cluster_arrive(); /* every CTA has begun before one writes to another */
    const T *in = static_cast<const T *>(p.logits) + (int64_t)b * p.logits_row;
    T *out = static_cast<T *>(p.out) + (int64_t)b * p.out_row;
    const uint32_t V = p.vocab;
    /* vectors are cut at 16-byte boundaries of the input row: vector i holds
     * the tokens i N - mis .. i N - mis + N - 1 */
    const uint32_t mis = kAligned ? 0u : (uint32_t)((reinterpret_cast<uintptr_t>(in) / sizeof(T)) % N);
    const bool wide_out = kAligned || ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    const uint32_t nvec = (mis + V + N - 1) / N;
    const uint32_t v0 = min(nvec, rank * p.slice_vecs), v1 = min(nvec, v0 + p.slice_vecs);
    const int32_t first = (int32_t)(v0 * N) - (int32_t)mis; /* token of the table's first count */
    const int32_t lo = max(first, 0), hi = min((int32_t)V, (int32_t)(v1 * N) - (int32_t)mis);
    const uint32_t *mask = p.mask == nullptr ? nullptr : p.mask + (int64_t)b * p.mask_row;
    const uint32_t size = (p.slice_vecs * N + 127) & ~127u; /* tokens of the table */
    uint32_t *past = table + size * sizeof(W) / 4, *biased = past + size / 32;

    int32_t *slice_id = reinterpret_cast<int32_t *>(biased + size / 32);
    float *slice_bias = reinterpret_cast<float *>(slice_id + p.biases);

    /* the vectors [va, vb) lie in the row whole */
    const uint32_t va = max(v0, mis != 0 ? 1u : 0u), vb = min(v1, nvec - ((mis + V) % N != 0 ? 1u : 0u));
    const uint4 *src = reinterpret_cast<const uint4 *>(in - mis);
    uint4 w[kUnroll];
    uint32_t allow[kUnroll];
    const uint8_t *mask8 = reinterpret_cast<const uint8_t *>(mask);
    /* N bits of vector i of a row of bits that starts with a vector's first token */
    auto bits_of = [](const uint8_t *bits, uint32_t i) {
        return N == 8 ? (uint32_t)bits[i] : (uint32_t)bits[i >> 1] >> (4 * (i & 1)) & 15u;
    };
    auto load = [&](uint32_t base) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const uint32_t i = base + u * kThreads;
            if (i < vb) {
                w[u] = __ldcs(src + i);
                if (mask != nullptr) {
                    const uint32_t e0 = i * N - mis;
                    allow[u] = mis == 0 ? bits_of(mask8, i)
                                        : __funnelshift_r(mask[e0 >> 5], mask[(e0 + N - 1) >> 5], e0 & 31);
                }
            }
        }
    };
    load(va + tid); /* on their way while the table is built */

    const uint32_t biases = p.bias_ids == nullptr ? 0 : p.biases;
    const int32_t *bias_ids = p.bias_ids + (int64_t)b * p.bias_ids_row;
    const int32_t len = p.tokens == nullptr ? 0 : p.lens == nullptr ? (int32_t)p.history : min(p.lens[b], (int32_t)p.history);
    const bool use_table = len > 0 || biases > 0;
    if (use_table) {
        const int32_t *ids = p.tokens + (int64_t)b * p.tokens_row;
        int32_t id[kHistoryUnroll];
        auto load_ids = [&](int32_t i0) {
#pragma unroll
            for (int u = 0; u < kHistoryUnroll; ++u) {
                const int32_t i = i0 + u * (int32_t)kThreads;
                id[u] = i < len ? ids[i] : -1;
            }
        };
        load_ids((int32_t)tid);
        /* warp 0 takes the biases, 64 at a time */
        const float *bias = p.bias + (int64_t)b * p.bias_row;
        int32_t bias_id[2];
        float bias_value[2];
        auto load_biases = [&](uint32_t i0) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t i = i0 + 32 * u + lane;
                bias_id[u] = i < biases ? bias_ids[i] : -1;
                bias_value[u] = i < biases ? bias[i] : 0.0f;
            }
        };
        if (warp == 0) load_biases(0);
        const int32_t made = p.prompt_lens == nullptr ? 0 : p.prompt_lens[b];
        const uint32_t clear = (size * sizeof(W) / 4 + size / 16) / 4;
        for (uint32_t i = tid; i < clear; i += kThreads) reinterpret_cast<uint4 *>(table)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        const uint32_t span = hi > lo ? (uint32_t)(hi - lo) : 0u;
        for (int32_t i0 = (int32_t)tid; i0 < len; i0 += (int32_t)kThreads * kHistoryUnroll) {
            if (i0 != (int32_t)tid) load_ids(i0);
#pragma unroll
            for (int u = 0; u < kHistoryUnroll; ++u) {
                if ((uint32_t)(id[u] - lo) >= span) continue;
                const uint32_t at = (uint32_t)(id[u] - first);
                atomicOr(&past[at >> 5], 1u << (at & 31));
                if (i0 + u * (int32_t)kThreads >= made) {
                    if (sizeof(W) == 4)
                        atomicAdd(&table[at], 1u);
                    else
                        atomicAdd(&table[at >> 1], (at & 1) ? 65536u : 1u); /* no count reaches 65536: nothing is carried */
                }
            }
        }
        if (warp == 0) {
            /* those of the slice, in list order */
            uint32_t found = 0;
            for (uint32_t i0 = 0; i0 < biases; i0 += 64) {
                if (i0 != 0) load_biases(i0);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const bool here = (uint32_t)(bias_id[u] - lo) < span;
                    const uint32_t who = __ballot_sync(0xffffffffu, here);
                    if (here) {
                        const uint32_t at = (uint32_t)(bias_id[u] - first), spot = found + __popc(who & ((1u << lane) - 1));
                        atomicOr(&biased[at >> 5], 1u << (at & 31));
                        slice_id[spot] = bias_id[u];
                        slice_bias[spot] = bias_value[u];
                    }
                    found += __popc(who);
                }
            }
            if (lane == 0) slice_biases = found;
        }
        __syncthreads();
    }

    if (use_table) {
        const float repetition = p.repetition == nullptr ? 1.0f : p.repetition[b];
        const float presence = p.presence == nullptr ? 0.0f : p.presence[b];
        const float frequency = p.frequency == nullptr ? 0.0f : p.frequency[b];
        /* 32 words of bits at a time: the set ones in order, one for each lane */
        for (uint32_t w0 = warp * 32; w0 < size / 32; w0 += kThreads) {
            const uint32_t i = w0 + lane, set = i < size / 32 ? past[i] | biased[i] : 0u;
            uint32_t upto = __popc(set);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t below = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= (uint32_t)o) upto += below;
            }
            const uint32_t total = __shfl_sync(0xffffffffu, upto, 31);
            for (uint32_t k0 = 0; k0 < total; k0 += 32) {
                const uint32_t k = k0 + lane;
                /* the word that the k-th set bit is in: the first whose running count exceeds k */
                uint32_t src = 0;
#pragma unroll
                for (uint32_t half = 16; half > 0; half >>= 1)
                    if (__shfl_sync(0xffffffffu, upto, src + half - 1) <= k) src += half;
                src &= 31;
                const uint32_t word = __shfl_sync(0xffffffffu, set, src), before = __shfl_sync(0xffffffffu, upto, src) - __popc(word);
                if (k >= total) continue;
                const uint32_t at = 32 * (w0 + src) + nth_bit(word, k - before);
                const int32_t id = first + (int32_t)at;
                const uint32_t n = sizeof(W) == 4 ? table[at] : (table[at >> 1] >> (16 * (at & 1))) & 0xFFFFu;
                float x = load_one(in + id);
                if ((past[at >> 5] >> (at & 31)) & 1u) x = x > 0.0f ? __fdiv_rn(x, repetition) : __fmul_rn(x, repetition);
                if (n != 0) x = __fsub_rn(__fsub_rn(x, __fmul_rn(frequency, (float)n)), presence);
                if ((biased[at >> 5] >> (at & 31)) & 1u) {
                    float sum = 0.0f;
                    bool any = false;
                    for (uint32_t e = 0; e < slice_biases; ++e)
                        if (slice_id[e] == id) {
                            sum = any ? __fadd_rn(sum, slice_bias[e]) : slice_bias[e];
                            any = true;
                        }
                    x = __fadd_rn(x, sum);
                }
                if (mask != nullptr && !((mask[id >> 5] >> (id & 31)) & 1u)) x = kNegInf;
                reinterpret_cast<W *>(table)[at] = (W)Vec<T>::bits(x);
            }
        }
        __syncthreads();
    }

    /* dense pass: the mask, the results of the tokens with a bit, and the largest */
    unsigned long long best = 0;
    float top = kNegInf;
    uint32_t top_vec = 0;
    const uint8_t *past8 = reinterpret_cast<const uint8_t *>(past), *biased8 = reinterpret_cast<const uint8_t *>(biased);
    auto own_bits = [&](uint32_t i) { return use_table ? bits_of(past8, i - v0) | bits_of(biased8, i - v0) : 0u; };
    auto edge = [&](uint32_t i) {
        /* a row's ragged first or last vector */
        const int32_t e0 = (int32_t)(i * N) - (int32_t)mis;
        const uint32_t own = own_bits(i);
        for (int32_t e = max(e0, 0); e < min(e0 + N, (int32_t)V); ++e) {
            float x = load_one(in + e);
            if ((own >> (e - e0)) & 1u)
                x = from_bits(reinterpret_cast<const W *>(table)[e - first], T());
            else if (mask != nullptr && !((mask[e >> 5] >> (e & 31)) & 1u))
                x = kNegInf;
            store_one(out + e, x);
            const unsigned long long key = pick_key(x, (uint32_t)e);
            best = key > best ? key : best;
        }
    };
    if (tid == 0 && v0 < min(va, v1)) edge(v0);
    if (tid == 32 && vb < v1 && v1 - 1 >= va) edge(v1 - 1);
    /* the table's words of vector i of the slice, as a vector */
    auto results = [&](uint32_t i) {
        const uint4 *t = reinterpret_cast<const uint4 *>(table);
        if (sizeof(W) == sizeof(T)) return t[i];
        const uint4 a = t[2 * i], c = t[2 * i + 1];
        return make_uint4(a.x | (a.y << 16), a.z | (a.w << 16), c.x | (c.y << 16), c.z | (c.w << 16));
    };
    /* the pass, for rows with and without a table and a mask */
    auto dense = [&](auto table_on, auto mask_on) {
        constexpr bool kTable = decltype(table_on)::value, kMask = decltype(mask_on)::value;
        auto one = [&](uint32_t i, uint4 o, uint32_t may) {
            const uint32_t own = kTable ? bits_of(past8, i - v0) | bits_of(biased8, i - v0) : 0u;
            if (kMask) o = Vec<T>::only(o, may);
            if (kTable && own) o = Vec<T>::blend(o, results(i - v0), own);
            if (wide_out) {
                __stcs(reinterpret_cast<uint4 *>(out - mis) + i, o);
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) store_one(out - mis + (i * N + j), Vec<T>::value(o, j));
            }
            const float m = Vec<T>::largest(o);
            if (m > top) {
                top = m;
                top_vec = i;
            }
        };
        for (uint32_t base = va + tid; base < vb; base += kThreads * kUnroll) {
            if (base != va + tid) load(base);
            if (base + (kUnroll - 1) * kThreads < vb) {
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) one(base + u * kThreads, w[u], allow[u]);
            } else {
#pragma unroll
                for (int u = 0; u < kUnroll - 1; ++u)
                    if (base + u * kThreads < vb) one(base + u * kThreads, w[u], allow[u]);
            }
        }
    };
    using std::bool_constant;
    if (use_table) {
        if (mask != nullptr)
            dense(bool_constant<true>(), bool_constant<true>());
        else
            dense(bool_constant<true>(), bool_constant<false>());
    } else {
        if (mask != nullptr)
            dense(bool_constant<false>(), bool_constant<true>());
        else
            dense(bool_constant<false>(), bool_constant<false>());
    }
    if (top > kNegInf) {
        /* this thread's own vector again: which of its tokens it was */
        const T *again = out - mis + (size_t)top_vec * N;
        uint32_t e = 0;
        while (e + 1 < N && load_one(again + e) != top) ++e;
        const unsigned long long key = pick_key(top, top_vec * N - mis + e);
        best = key > best ? key : best;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
    }
    if (lane == 0) warp_key[warp] = best;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (uint32_t i = 1; i < kThreads / 32; ++i) best = warp_key[i] > best ? warp_key[i] : best;
    }
    cluster_wait();
    if (tid == 0) cluster.map_shared_rank(slice_key, 0)[rank] = best;
    cluster_arrive();
    if (rank != 0) return;
    cluster_wait();
    if (tid == 0) {
        for (uint32_t c = 0; c < C; ++c) best = slice_key[c] > best ? slice_key[c] : best;
        p.picks[b] = (uint32_t)(best >> 32) > kKeyNegInf ? (int32_t)(0xFFFFFFFFu - (uint32_t)best) : -1;
    }
}

/* The largest table: a row of kMaxVocab tokens in kMaxCluster slices. Every
 * call sets this one limit, so that calls of other threads and calls captured
 * into a graph before keep theirs. */
template <typename T, typename W>
constexpr size_t max_smem() {
    constexpr size_t N = Vec<T>::kN, vecs = (kMaxVocab + N - 1) / N + 1, size = ((vecs + kMaxCluster - 1) / kMaxCluster * N + 127) & ~(size_t)127;
    return size * sizeof(W) + size / 4 + 8 * (size_t)kMaxBiases;
}

template <typename T, typename W, bool kAligned>
cudaError_t launch_logits_t(LogitsParams &p, int sms, cudaStream_t stream) {
    constexpr uint32_t N = Vec<T>::kN;
    const uint32_t nvec = (p.vocab + N - 1) / N + 1; /* a row that starts inside a vector has one more */
    /* Slices: two CTAs for each SM, and a table of at most 32 KB, so that five
     * fit, as far as eight slices go (FP32 rows of more than 65536 tokens have
     * up to 128 KB). 256 rows of 32000: FP32 32 us with four slices, 40 with two; BF16 23 with
     * four, 19 with two. 100 rows FP32: 16.5 with eight, 11.6 with four. */
    uint32_t C = 1;
    while (C < kMaxCluster && (p.rows * C < 2u * (uint32_t)sms || nvec * N / C * sizeof(W) > 32768u + 64)) C *= 2;
    p.slice_vecs = (nvec + C - 1) / C;
    const bool use_table = p.tokens != nullptr || p.bias_ids != nullptr;
    const size_t size = (p.slice_vecs * N + 127) & ~(size_t)127;
    const size_t smem = use_table ? size * sizeof(W) + size / 4 + 8 * (size_t)p.biases : 0;
    static_assert(max_smem<T, W>() <= 227 * 1024 - 1024, "the largest table");
    cudaError_t e = cudaFuncSetAttribute(logits_kernel<T, W, kAligned>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)max_smem<T, W>());
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.rows * C);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, logits_kernel<T, W, kAligned>, p);
}

}  // namespace

cudaError_t launch_logits(LogitsParams p, bool bf16, int sms, cudaStream_t stream) {
    const int64_t per = bf16 ? 8 : 4;
    const bool aligned = ((reinterpret_cast<uintptr_t>(p.logits) | reinterpret_cast<uintptr_t>(p.out)) & 15) == 0 &&
                         (p.rows == 1 || (p.logits_row % per == 0 && p.out_row % per == 0));
    auto *launch = aligned ? launch_logits_t<float, uint32_t, true> : launch_logits_t<float, uint32_t, false>;
    if (bf16)
        launch = p.history > 65535u
                     ? aligned ? launch_logits_t<__nv_bfloat16, uint32_t, true> : launch_logits_t<__nv_bfloat16, uint32_t, false>
                 : aligned ? launch_logits_t<__nv_bfloat16, uint16_t, true>
                           : launch_logits_t<__nv_bfloat16, uint16_t, false>;
    return launch(p, sms, stream);
}

}  // namespace ops
}  // namespace gdn
