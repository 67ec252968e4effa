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
 * FP32; the state stays in registers over all tokens of the sequence. Measured
 * with BF16 heads of 256 x 256: one stream of 8 heads 3.7 us, 16 streams 13.0 us
 * (5.2 TB/s of state); the pipeline below takes over from there: 64 streams 49
 * us (5.5 TB/s), 256 streams 176 us (6.1 TB/s, 0.94 of a copy's).
 */
#include "gdn_ops.h"

#include <cuda_bf16.h>

namespace gdn {
namespace ops {

namespace {

constexpr int kLanesPerRow = 8;
/* 16 rows a CTA: five of them share an SM with heads of 256 (64 streams of two
 * tokens 64 us, with 32 rows 80, with 8 rows 70) */
constexpr int kStepThreads = 128;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void store_out(float *p, float x) { *p = x; }
__device__ __forceinline__ void store_out(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

/* One token on one row of S, of which this lane holds kVec float4: advances it
 * and returns the row's output (in all eight lanes). */
template <int kVec>
__device__ __forceinline__ float advance(float4 (&s)[kVec], const float4 *q4, const float4 *k4, float decay, float beta,
                                         float qk, float v) {
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
    const float delta = beta * (v - decay * r);
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
        const float4 a = k4[j * kLanesPerRow];
        s[j].x = fmaf(decay, s[j].x, a.x * delta);
        s[j].y = fmaf(decay, s[j].y, a.y * delta);
        s[j].z = fmaf(decay, s[j].z, a.z * delta);
        s[j].w = fmaf(decay, s[j].w, a.w * delta);
    }
    return decay * pq + qk * delta;
}

/* Tokens that no sequence covers give zeros: the rows of out before the
 * first and after the last sequence. `at` of `of` threads. */
template <typename T>
__device__ __forceinline__ void zero_uncovered(const DeltaParams &p, uint32_t at, uint32_t of) {
    T *out = static_cast<T *>(p.out);
    const Covered c = covered_tokens(p);
    const uint32_t width = p.HV * p.V;
    for (uint32_t t = c.first_outside(); t < p.tokens; t = c.next_outside(t))
        for (uint32_t i = at; i < width; i += of)
            store_out(out + (int64_t)t * p.out_token + (int64_t)(i / p.V) * p.out_head + i % p.V, 0.0f);
}

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
        zero_uncovered<T>(p, rem * blockDim.x + tid, p.HV * blocks * blockDim.x);
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
            const float o = advance<kVec>(s, q4, k4, dec[i], bet[i], alp[i], vs[i][tid / kLanesPerRow]);
            if (l8 == 0)
                store_out(out + (int64_t)(tile + i) * p.out_token + (int64_t)h * p.out_head + row, o);
        }
    }
#pragma unroll
    for (int j = 0; j < kVec; ++j) S[j * kLanesPerRow] = s[j];
}

/* ------------------------------------------------- many states: a pipeline
 *
 * With many states the kernel above is held up by its own phases (a CTA loads,
 * computes and stores in turn, and five CTAs fill an SM's registers): 5.4 TB/s
 * for 256 streams, against 6.1.
 * Here one CTA per SM walks a contiguous range of row blocks (up to 32 KB of
 * state each) through a ring in shared memory: one thread issues the bulk
 * copies in, eight warps advance a block in place, one thread issues the bulk
 * copy out. Three more warps stage the tokens' vectors ahead. */

constexpr int kRing = 4;                  /* row blocks in flight (256 streams: 3 197, 4 177, 5 189, 6 193 us) */
constexpr uint32_t kBlockBytes = 32768;
constexpr int kItems = 3, kItemTokens = 8; /* staged token groups, tokens of one */
constexpr int kRowThreads = 256;
constexpr int kPipeThreads = (9 + kItems) * 32; /* 8 warps of rows, the copies, one for each staged group */
constexpr uint64_t kWaitNs = 2000000000ull;

/* set when a wait of the pipeline ran out; read and cleared by the host */
__device__ int g_step_status;

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint64_t gtimer() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(20000u)
        : "memory");
    return ok != 0;
}
/* Bounded wait; false when the CTA gives up (here or elsewhere). */
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile uint32_t *abort) {
    if (mbar_try(bar, parity)) return true;
    const uint64_t t0 = gtimer();
    while (!mbar_try(bar, parity)) {
        if (*abort) return false;
        if (gtimer() - t0 > kWaitNs) {
            *abort = 1;
            atomicExch(&g_step_status, 1);
            return false;
        }
    }
    return true;
}
/* the same for a whole warp, with one answer */
__device__ __forceinline__ bool wait_bar_warp(uint32_t bar, uint32_t parity, volatile uint32_t *abort) {
    return __all_sync(0xffffffffu, wait_bar(bar, parity, abort));
}
/* AND of v over the threads of the row warps, which all wait for it: where
 * one of their waits ran out, all of them learn it at their next barrier,
 * whichever that is for each, and leave */
__device__ __forceinline__ bool rows_all(bool v) {
    uint32_t r;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.red.and.pred q, 1, %2, p;\n selp.u32 %0, 1, 0, q;\n}\n"
        : "=r"(r)
        : "r"((uint32_t)v), "r"(kRowThreads)
        : "memory");
    return r != 0;
}

/* What one row block is, written by the copying thread with its copy. */
struct BlockMeta {
    uint64_t state;            /* address of the rows */
    uint32_t t0, t1, h, row0;
    uint32_t item;             /* number of its first token group */
    uint32_t flags;
};
enum { kMetaEnd = 1, kMetaZero = 2, kMetaFresh = 4, kMetaLast = 8 };

struct Pipe {
    uint32_t rows, blocks;     /* rows of a block, blocks of a head */
    uint32_t units;            /* row blocks of all sequences and heads */
};

/* Row blocks [u0, u1) of a CTA as (sequence, head, block), in order. */
struct Walk {
    uint32_t u, n, h, blk, t0, t1;
    int64_t slot;
    bool fresh;
    __device__ __forceinline__ void read(const DeltaParams &p) {
        sequence_tokens(p, n, t0, t1);
        slot = sequence_slot(p, n);
        fresh = p.fresh != nullptr && p.fresh[n] != 0;
    }
    __device__ __forceinline__ Walk(const DeltaParams &p, const Pipe &g, uint32_t first) : u(first) {
        const uint32_t per = p.HV * g.blocks;
        n = u / per;
        h = (u - n * per) / g.blocks;
        blk = u - n * per - h * g.blocks;
        read(p);
    }
    __device__ __forceinline__ void next(const DeltaParams &p, const Pipe &g, uint32_t end) {
        ++u;
        if (++blk < g.blocks) return;
        blk = 0;
        if (++h < p.HV) return;
        h = 0;
        ++n;
        if (u < end) read(p);
    }
    __device__ __forceinline__ uint32_t tokens() const { return t1 - t0; }
    /* a state that neither changes nor gives outputs */
    __device__ __forceinline__ bool idle() const { return t0 == t1 && (slot < 0 || !fresh); }
};

template <int K>
struct PipeSmem {
    static constexpr uint32_t kQ = 0, kK = kItemTokens * K * 4, kV = 2 * kK, kScal = kV + kItemTokens * 256 * 4;
    static constexpr uint32_t kItem = kScal + kItemTokens * 16;
    static constexpr uint32_t kItemAt = kRing * kBlockBytes;
    static constexpr uint32_t kMeta = kItemAt + kItems * kItem;
    static constexpr uint32_t kBars = kMeta + kRing * sizeof(BlockMeta);
    static constexpr uint32_t kBytes = kBars + 8 * (2 * kRing + 2 * kItems) + 16 + 128;
};

template <int K, typename T>
__global__ void __launch_bounds__(kPipeThreads, 1) delta_pipe_kernel(const __grid_constant__ DeltaParams p,
                                                                     const __grid_constant__ Pipe g) {
    using L = PipeSmem<K>;
    constexpr int kVec = K / kLanesPerRow / 4;
    extern __shared__ uint8_t raw[];
    uint8_t *sm = raw + ((128u - (smem_u32(raw) & 127u)) & 127u);
    const uint32_t base = smem_u32(sm);
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t full = base + L::kBars, empty = full + 8 * kRing, item_full = empty + 8 * kRing,
                   item_empty = item_full + 8 * kItems;
    BlockMeta *meta = reinterpret_cast<BlockMeta *>(sm + L::kMeta);
    volatile uint32_t *abort = reinterpret_cast<volatile uint32_t *>(sm + L::kBars + 8 * (2 * kRing + 2 * kItems));
    /* a state is not wanted again before all the others have been */
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    const uint32_t u0 = (uint32_t)(((uint64_t)blockIdx.x * g.units) / gridDim.x);
    const uint32_t u1 = (uint32_t)(((uint64_t)(blockIdx.x + 1) * g.units) / gridDim.x);
    T *out = static_cast<T *>(p.out);
    if (tid == 0) {
        for (int i = 0; i < kRing; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < kItems; ++i) {
            mbar_init(item_full + 8 * i, 1);
            mbar_init(item_empty + 8 * i, 1);
        }
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();

    if (warp == 8) {
        if (lane == 0) {
            uint32_t i = 0, item = 0;
            const uint32_t bytes = g.rows * K * 4;
            for (Walk w(p, g, u0); w.u < u1; w.next(p, g, u1)) {
                if (w.idle()) continue;
                const uint32_t sl = i % kRing;
                if (i >= kRing && !wait_bar(empty + 8 * sl, (i / kRing - 1) & 1u, abort)) break;
                BlockMeta m;
                m.t0 = w.t0;
                m.t1 = w.t1;
                m.h = w.h;
                m.row0 = w.blk * g.rows;
                m.item = item;
                float *S = p.state + (w.slot < 0 ? 0 : w.slot * p.state_slot) + ((int64_t)w.h * p.V + m.row0) * K;
                m.state = reinterpret_cast<uint64_t>(S);
                /* a group of few tokens serves all of the head's blocks here, a longer sequence is staged block by block */
                const bool shared = w.tokens() <= (uint32_t)kItemTokens;
                const bool last = !shared || w.blk + 1 == g.blocks || w.u + 1 == u1;
                m.flags = (w.slot < 0 ? kMetaZero : 0) | (w.fresh ? kMetaFresh : 0) | (last ? kMetaLast : 0);
                if (w.slot >= 0 && last) item += (w.tokens() + kItemTokens - 1) / kItemTokens;
                meta[sl] = m;
                if (w.slot >= 0 && !w.fresh) {
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full + 8 * sl), "r"(bytes)
                                 : "memory");
                    if (w.u + 1 != p.drop)
                        asm volatile(
                            "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
                                base + sl * kBlockBytes),
                            "l"(S), "r"(bytes), "r"(full + 8 * sl), "l"(policy)
                            : "memory");
                } else {
                    mbar_arrive(full + 8 * sl);
                }
                ++i;
            }
            /* copies under way land before the CTA ends (an abort does not stop them) */
            for (uint32_t j = i > kRing ? i - kRing : 0; j < i; ++j) {
                const uint64_t w0 = gtimer();
                while (!mbar_try(full + 8 * (j % kRing), (j / kRing) & 1u) && gtimer() - w0 < kWaitNs) {
                }
            }
            const uint32_t sl = i % kRing;
            if (i < kRing || wait_bar(empty + 8 * sl, (i / kRing - 1) & 1u, abort)) {
                meta[sl].flags = kMetaEnd;
                mbar_arrive(full + 8 * sl);
            }
        }
        return;
    }
    if (warp > 8) {
        /* token groups: warp 9 + j takes the groups j, j + kItems, ... */
        const T *q = static_cast<const T *>(p.q), *k = static_cast<const T *>(p.k), *v = static_cast<const T *>(p.v);
        uint32_t item = 0;
        for (Walk w(p, g, u0); w.u < u1; w.next(p, g, u1)) {
            if (w.idle() || w.slot < 0) continue;
            const bool shared = w.tokens() <= (uint32_t)kItemTokens;
            if (shared && !(w.blk + 1 == g.blocks || w.u + 1 == u1)) continue;
            const uint32_t hq = w.h / (p.HV / p.H);
            for (uint32_t tile = w.t0; tile < w.t1; tile += kItemTokens, ++item) {
                if (item % kItems != warp - 9) continue;
                const uint32_t sl = item % kItems, nt = min((uint32_t)kItemTokens, w.t1 - tile);
                float *qs = reinterpret_cast<float *>(sm + L::kItemAt + sl * L::kItem + L::kQ);
                float *ks = reinterpret_cast<float *>(sm + L::kItemAt + sl * L::kItem + L::kK);
                float *vs = reinterpret_cast<float *>(sm + L::kItemAt + sl * L::kItem + L::kV);
                float *sc = reinterpret_cast<float *>(sm + L::kItemAt + sl * L::kItem + L::kScal);
                for (uint32_t i = 0; i < nt; ++i) {
                    const int64_t t = tile + i;
                    const T *qt = q + t * p.q_token + (int64_t)hq * p.q_head, *kt = k + t * p.k_token + (int64_t)hq * p.k_head;
                    const T *vt = v + t * p.v_token + (int64_t)w.h * p.v_head;
                    float qv[K / 32], kv[K / 32], vv[8], qq = 0.f, kk = 0.f, qk = 0.f;
#pragma unroll
                    for (int j = 0; j < K / 32; ++j) {
                        qv[j] = to_float(qt[lane + 32 * j]);
                        kv[j] = to_float(kt[lane + 32 * j]);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) vv[j] = lane + 32 * j < p.V ? to_float(vt[lane + 32 * j]) : 0.f;
                    const float gv = p.g[t * p.g_token + (int64_t)w.h * p.g_head];
                    const float bv = p.beta[t * p.beta_token + (int64_t)w.h * p.beta_head];
#pragma unroll
                    for (int j = 0; j < K / 32; ++j) {
                        qq = fmaf(qv[j], qv[j], qq);
                        kk = fmaf(kv[j], kv[j], kk);
                        qk = fmaf(qv[j], kv[j], qk);
                    }
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) {
                        qq += __shfl_xor_sync(0xffffffffu, qq, o);
                        kk += __shfl_xor_sync(0xffffffffu, kk, o);
                        qk += __shfl_xor_sync(0xffffffffu, qk, o);
                    }
                    const float qi = p.normalize ? p.scale / sqrtf(qq + 1e-6f) : p.scale;
                    const float ki = p.normalize ? 1.0f / sqrtf(kk + 1e-6f) : 1.0f;
                    if (i == 0 && item >= kItems &&
                        !wait_bar_warp(item_empty + 8 * sl, (item / kItems - 1) & 1u, abort))
                        return;
#pragma unroll
                    for (int j = 0; j < K / 32; ++j) {
                        qs[i * K + lane + 32 * j] = qv[j] * qi;
                        ks[i * K + lane + 32 * j] = kv[j] * ki;
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) vs[i * 256 + lane + 32 * j] = vv[j];
                    if (lane == 0) *reinterpret_cast<float4 *>(sc + 4 * i) = make_float4(expf(gv), bv, qk * qi * ki, 0.f);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(item_full + 8 * sl);
            }
        }
        return;
    }
    if (p.starts != nullptr && blockIdx.x + 1 == gridDim.x) zero_uncovered<T>(p, tid, kRowThreads);
    /* rows: eight lanes each, 32 rows at a time */
    const uint32_t r8 = tid / kLanesPerRow, l8 = tid & (kLanesPerRow - 1);
    bool go = true;
    for (uint32_t i = 0; go; ++i) {
        const uint32_t sl = i % kRing;
        bool ok = wait_bar_warp(full + 8 * sl, (i / kRing) & 1u, abort);
        BlockMeta m;
        if (ok) m = meta[sl];
        ok = ok && !(m.flags & kMetaEnd);
        const bool has_state = ok && !(m.flags & kMetaZero);
        float *rows = reinterpret_cast<float *>(sm + sl * kBlockBytes);
        if (ok && !has_state)
            for (uint32_t t = m.t0; t < m.t1; ++t)
                for (uint32_t r = tid; r < g.rows; r += kRowThreads)
                    store_out(out + (int64_t)t * p.out_token + (int64_t)m.h * p.out_head + m.row0 + r, 0.0f);
        const uint32_t groups = has_state ? (m.t1 - m.t0 + kItemTokens - 1) / kItemTokens : 0;
        if (has_state && groups == 0)
            for (uint32_t j = tid; j < g.rows * K / 4; j += kRowThreads)
                reinterpret_cast<float4 *>(rows)[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint32_t gi = 0; ok && gi < groups; ++gi) {
            const uint32_t item = m.item + gi, is = item % kItems;
            ok = wait_bar_warp(item_full + 8 * is, (item / kItems) & 1u, abort);
            if (!ok) break;
            const uint8_t *it = sm + L::kItemAt + is * L::kItem;
            const uint32_t nt = min((uint32_t)kItemTokens, m.t1 - m.t0 - gi * kItemTokens);
            const bool zero = gi == 0 && (m.flags & kMetaFresh);
            for (uint32_t r = r8; r < g.rows; r += kRowThreads / kLanesPerRow) {
                float4 *S = reinterpret_cast<float4 *>(rows + r * K) + l8;
                float4 s[kVec];
#pragma unroll
                for (int j = 0; j < kVec; ++j) s[j] = zero ? make_float4(0.f, 0.f, 0.f, 0.f) : S[j * kLanesPerRow];
                for (uint32_t t = 0; t < nt; ++t) {
                    const float4 *k4 = reinterpret_cast<const float4 *>(it + L::kK) + t * (K / 4) + l8;
                    const float4 *q4 = reinterpret_cast<const float4 *>(it + L::kQ) + t * (K / 4) + l8;
                    const float4 sc = *reinterpret_cast<const float4 *>(it + L::kScal + 16 * t);
                    const float vv = reinterpret_cast<const float *>(it + L::kV)[t * 256 + m.row0 + r];
                    const float o = advance<kVec>(s, q4, k4, sc.x, sc.y, sc.z, vv);
                    if (l8 == 0)
                        store_out(out + (int64_t)(m.t0 + gi * kItemTokens + t) * p.out_token + (int64_t)m.h * p.out_head +
                                      m.row0 + r, o);
                }
#pragma unroll
                for (int j = 0; j < kVec; ++j) S[j * kLanesPerRow] = s[j];
            }
            if (gi + 1 < groups) {
                /* a longer sequence's group is done with here */
                go = rows_all(true);
                if (!go) break;
                if (tid == 0) mbar_arrive(item_empty + 8 * is);
            }
        }
        if (!go) break;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        go = rows_all(ok); /* not at the end, nor where a wait ran out */
        if (go && tid == 0) {
            if (has_state) {
                if (groups != 0 && (m.flags & kMetaLast)) mbar_arrive(item_empty + 8 * ((m.item + groups - 1) % kItems));
                asm volatile("cp.async.bulk.global.shared::cta.bulk_group.L2::cache_hint [%0], [%1], %2, %3;" ::"l"(m.state),
                             "r"(base + sl * kBlockBytes), "r"(g.rows * K * 4), "l"(policy)
                             : "memory");
            }
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            /* the block before this one has left shared memory: its place is free */
            asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            if (i > 0) mbar_arrive(empty + 8 * ((i - 1) % kRing));
        }
    }
    if (tid == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    if (!rows_all(*abort == 0)) {
        /* given up: none of this CTA's states is left that could pass for one */
        const float bad = __int_as_float(0x7fc00000);
        for (Walk w(p, g, u0); w.u < u1; w.next(p, g, u1)) {
            if (w.idle() || w.slot < 0) continue;
            float4 *S = reinterpret_cast<float4 *>(p.state + w.slot * p.state_slot + ((int64_t)w.h * p.V + w.blk * g.rows) * K);
            for (uint32_t j = tid; j < g.rows * K / 4; j += kRowThreads) S[j] = make_float4(bad, bad, bad, bad);
        }
    }
}

template <int K>
cudaError_t launch_step_k(const DeltaParams &p, bool bf16, int sms, cudaStream_t stream) {
    /* The pipeline for one token a sequence (on average at most), from eight
     * row blocks per SM on, where it has filled: 20 streams of 8 heads of 256 x
     * 256 18.1 us against 18.4, 64 streams 49 against 56, 256 of 8 heads of 128
     * x 128 50 against 56. Not for heads of 64 x 64, a block each (256 of 8
     * heads 19.6 against 18.5), nor for more tokens: sequences of very
     * different lengths suit the kernel whose CTAs end on their own (256
     * streams of 12 heads of 128 x 128 with 0 to 6 tokens 188 against 99). */
    if constexpr (K >= 128) {
        Pipe g;
        g.rows = 32;
        for (uint32_t r = 64; r <= p.V && r * K * 4 <= kBlockBytes; r += 32)
            if (p.V % r == 0) g.rows = r;
        g.blocks = p.V / g.rows;
        g.units = p.N * p.HV * g.blocks;
        if (g.units >= 8u * (uint32_t)sms && p.tokens <= p.N) {
            auto *kernel = bf16 ? delta_pipe_kernel<K, __nv_bfloat16> : delta_pipe_kernel<K, float>;
            cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PipeSmem<K>::kBytes);
            if (e != cudaSuccess) return e;
            return launch(kernel, dim3(sms), kPipeThreads, PipeSmem<K>::kBytes, stream, p, g);
        }
    }
    const uint32_t rows = kStepThreads / kLanesPerRow;
    const uint32_t grid = (p.N + (p.starts != nullptr ? 1u : 0u)) * p.HV * (p.V / rows);
    return launch(bf16 ? delta_step_kernel<K, __nv_bfloat16> : delta_step_kernel<K, float>, dim3(grid), kStepThreads, 0, stream, p);
}

}  // namespace

cudaError_t launch_delta_step(const DeltaParams &p, bool bf16, int sms, cudaStream_t stream) {
    switch (p.K) {
        case 64: return launch_step_k<64>(p, bf16, sms, stream);
        case 128: return launch_step_k<128>(p, bf16, sms, stream);
        default: return launch_step_k<256>(p, bf16, sms, stream);
    }
}

cudaError_t delta_step_status(int *status) {
    cudaError_t e = cudaMemcpyFromSymbol(status, g_step_status, sizeof(int));
    const int zero = 0;
    if (e == cudaSuccess && *status != 0) e = cudaMemcpyToSymbol(g_step_status, &zero, sizeof(int));
    return e;
}

}  // namespace ops
}  // namespace gdn
