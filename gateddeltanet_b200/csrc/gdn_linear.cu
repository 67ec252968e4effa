/* gdn_linear.cu -- y = act(sx sw x W^T + bias) + residual on the tcgen05
 * tensor cores, for more tokens than gdn_linear_few.cu takes.
 *
 * D [tokens][rows of W] is cut into tiles of 128 tokens by up to 256 rows, or,
 * with two CTAs to a tile (cta_group::2), of 256 tokens: each of the two then
 * loads 128 tokens and half of the rows of W, which is what lets L2 keep up with
 * the tensor cores. BF16 operands go to kind::f16 and 8-bit ones to
 * kind::f8f6f4; both come as blocks of 128 bytes of k in the 128-byte swizzle,
 * so that the two differ in the instruction alone. Sums are FP32 in TMEM. For
 * swiglu a tile holds the same outputs of both halves of W side by side.
 *
 * A CTA has one warp that starts the TMA copies into a ring of stages, one
 * that starts the MMAs, and eight that take finished sums from TMEM to memory
 * (scales, bias, activation, residual) while the next tile's MMAs run: there
 * are two accumulators. CTAs walk over the tiles, tokens first.
 *
 * Where there are too few tiles for all SMs, the CTAs of a cluster divide k:
 * each one's sums go to its shared memory, and each adds up, in the order of
 * the cluster's ranks, a part of the columns from all of them.
 *
 * Every wait is bounded (2 s). A CTA whose wait ran out writes NaN to its
 * outputs and sets g_linear_status.
 */
#include "gdn_linear.h"

#include <cuda.h>

#include <atomic>

namespace gdn {
namespace ops {

namespace {

constexpr uint64_t kWaitNs = 2000000000ull;
constexpr uint32_t kEpilogueWarps = 8;
constexpr uint32_t kLinearThreads = (kEpilogueWarps + 2) * 32;
constexpr uint32_t kBlock = 128;                  /* bytes of k in a stage */
constexpr uint32_t kRowsA = 128;                  /* tokens of a CTA */
constexpr uint32_t kBytesA = kRowsA * kBlock;
constexpr uint32_t kMaxStages = 8;
constexpr uint32_t kMaxN = 256;

/* set when a wait of a kernel ran out; read and cleared by the host */
__device__ int g_linear_status;

/* a launch's tiles */
struct LinearShape {
    uint32_t n;        /* columns of a tile (rows of W): a multiple of 16, of 32 with two CTAs or for swiglu */
    uint32_t outs;     /* outputs of a tile: n, or n / 2 for swiglu */
    uint32_t split;    /* CTAs that divide k (one CTA to a tile), or 1 */
    uint32_t stages;
    uint32_t rows_a;   /* rows of a copy of x: 128, or fewer where there are fewer tokens */
    uint32_t tiles_m, tiles_n, blocks; /* blocks: of k */
    uint32_t columns;  /* of TMEM */
};

struct SharedTail {
    uint64_t full[kMaxStages], empty[kMaxStages], sums_full[2], sums_empty[2], drain;
    uint32_t tmem, abort, failed;
    float scale[2][kMaxN], bias[2][kMaxN]; /* of an accumulator's columns */
};

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint64_t gtimer() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
/* at a barrier of any CTA of the cluster */
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(20000u)
        : "memory");
    return ok != 0;
}
/* Bounded wait; false when the CTA gives up (here or elsewhere). */
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile uint32_t *abort) {
    if (mbar_try(bar, parity)) return true;
    const uint64_t t0 = gtimer();
    while (true) {
#pragma unroll 1
        for (int i = 0; i < 16; ++i)
            if (mbar_try(bar, parity)) return true;
        if (*abort) return false;
        if (gtimer() - t0 > kWaitNs) {
            *abort = 1;
            atomicExch(&g_linear_status, 1);
            return false;
        }
    }
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
/* a shared address of CTA `rank` of the cluster */
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 load_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t load_cluster(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

/* K-major operand in the 128-byte swizzle: start >> 4 (bits 0-13), leading
 * offset (16-29, not used), 1 KB from eight rows to the next (32-45), version 1
 * (46-47), layout 2 (61-63). */
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
/* D FP32 (bits 4-5 = 1); A and B (7-9, 10-12): BF16 is 1 of kind::f16, E4M3 0 of kind::f8f6f4; N >> 3 at 17, M >> 4 at 24 */
template <bool kFp8>
__device__ __forceinline__ uint32_t instr_desc(uint32_t m, uint32_t n) {
    return (1u << 4) | (kFp8 ? 0u : (1u << 7) | (1u << 10)) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

template <int kCtas, bool kFp8>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
#define GDN_MMA(GROUP, KIND)                                                                                      \
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::" GROUP ".kind::" KIND        \
                 " [%0], %1, %2, %3, p;\n}\n" ::"r"(d),                                                            \
                 "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)                                             \
                 : "memory")
    if constexpr (kCtas == 1 && !kFp8) GDN_MMA("1", "f16");
    if constexpr (kCtas == 1 && kFp8) GDN_MMA("1", "f8f6f4");
    if constexpr (kCtas == 2 && !kFp8) GDN_MMA("2", "f16");
    if constexpr (kCtas == 2 && kFp8) GDN_MMA("2", "f8f6f4");
#undef GDN_MMA
}
/* arrives at the barrier (of both CTAs of a pair) when the MMAs started so far have ended */
template <int kCtas>
__device__ __forceinline__ void commit(uint32_t bar) {
    if constexpr (kCtas == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                     "h"((uint16_t)3)
                     : "memory");
}
/* a box at (k, row); with two CTAs the barrier may be the other one's */
template <int kCtas>
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap *map, uint32_t k, uint32_t row, uint32_t bar) {
    if constexpr (kCtas == 1)
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                     "l"(map), "r"(k), "r"(row), "r"(bar)
                     : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
            "l"(map), "r"(k), "r"(row), "r"(bar)
            : "memory");
}
/* 16 FP32 columns of this thread's TMEM lane; tc_wait before the values are used */
__device__ __forceinline__ void tc_ld16(uint32_t addr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tc_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kEpilogueWarps * 32) : "memory"); }

/* Columns c .. c + 15 of the tile (of its outputs) of one token to memory: v the sums, up
 * those of the second half for swiglu. `scale` and `bias` are those of the tile's
 * columns, with the second half's at g.outs. */
struct Row {
    uint32_t token, n; /* n: the output of column c */
    float scale;
};
__device__ __forceinline__ void finish16(const LinearParams &p, const Row &r, float (&v)[16], float (&up)[16], const float *scale,
                                         const float *bias, uint32_t outs, bool wide_out, bool wide_res) {
    const bool pairs = p.activation == kSwiglu;
    if (p.type == kE4M3) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            v[i] *= r.scale * scale[i];
            if (pairs) up[i] *= r.scale * scale[outs + i];
        }
    }
    if (p.bias != nullptr) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            v[i] += bias[i];
            if (pairs) up[i] += bias[outs + i];
        }
    }
    if (p.activation != kNoActivation) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = activate(p.activation, v[i], up[i]);
    }
    const bool whole = r.n + 16 <= p.outputs;
    if (p.residual != nullptr) {
        const int64_t at = r.token * p.residual_row + r.n;
        if (whole && wide_res) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float e[8];
                load8(p.residual, at + 8 * h, p.residual_type, e);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[8 * h + i] += e[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (r.n + i < p.outputs) v[i] += load1(p.residual, at + i, p.residual_type);
        }
    }
    const int64_t at = r.token * p.out_row + r.n;
    if (whole && wide_out) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = v[8 * h + i];
            store8(p.out, at + 8 * h, p.out_type, e);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (r.n + i < p.outputs) store1(p.out, at + i, p.out_type, v[i]);
    }
}

template <int kCtas, bool kFp8>
__global__ void __launch_bounds__(kLinearThreads, 1)
    linear_kernel(const __grid_constant__ LinearParams p, const __grid_constant__ CUtensorMap map_x,
                  const __grid_constant__ CUtensorMap map_w, const LinearShape g) {
    extern __shared__ uint8_t raw[];
    constexpr uint32_t kElem = kFp8 ? 1 : 2;
    const uint32_t start = (smem_u32(raw) + 1023u) & ~1023u;
    uint8_t *base = raw + (start - smem_u32(raw));
    const uint32_t bytes_b = g.n / kCtas * kBlock, stage = kBytesA + bytes_b;
    SharedTail *s = reinterpret_cast<SharedTail *>(base + g.stages * stage);
    volatile uint32_t *abort = &s->abort;
    const uint32_t full = smem_u32(s->full), empty = smem_u32(s->empty), sums_full = smem_u32(s->sums_full),
                   sums_empty = smem_u32(s->sums_empty), drain = smem_u32(&s->drain);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = kCtas == 1 && g.split == 1 ? 0 : cluster_rank(), pair = kCtas == 2 ? rank : 0;
    const uint32_t group = kCtas * g.split, worker = blockIdx.x / group, workers = gridDim.x / group;
    const uint32_t tiles = g.tiles_m * g.tiles_n;
    const uint32_t b0 = kCtas == 1 ? (uint32_t)((uint64_t)g.blocks * rank / g.split) : 0;
    const uint32_t b1 = kCtas == 1 ? (uint32_t)((uint64_t)g.blocks * (rank + 1) / g.split) : g.blocks;
    const bool pairs = p.activation == kSwiglu;

    if (tid == 0) {
        for (uint32_t i = 0; i < g.stages; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(sums_full + 8 * i, 1);
            mbar_init(sums_empty + 8 * i, kCtas * kEpilogueWarps);
        }
        mbar_init(drain, 1);
        s->abort = 0;
        s->failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        if constexpr (kCtas == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s->tmem)), "r"(g.columns) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s->tmem)), "r"(g.columns) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if (kCtas == 2) cluster_sync(); /* the other CTA's barriers are ready */
    tc_fence_after();
    const uint32_t tmem = s->tmem, second = g.columns / 2; /* columns from one accumulator to the other */

    if (warp == kEpilogueWarps) {
        if (lane == 0) {
            const uint32_t bar0 = kCtas == 2 ? map_rank(full, 0) : full; /* the pair's MMAs wait at the first CTA's */
            const uint32_t bytes = kCtas * (g.rows_a * kBlock + bytes_b);
            uint32_t it = 0;
            bool ok = true;
            for (uint32_t tile = worker; ok && tile < tiles; tile += workers) {
                const uint32_t m0 = (tile % g.tiles_m * kCtas + pair) * kRowsA, n0 = tile / g.tiles_m * g.outs;
                for (uint32_t b = b0; b < b1; ++b, ++it) {
                    const uint32_t slot = it % g.stages;
                    if (it >= g.stages && !wait_bar(empty + 8 * slot, (it / g.stages - 1) & 1u, abort)) {
                        ok = false;
                        break;
                    }
                    if (pair == 0) mbar_expect_tx(full + 8 * slot, bytes);
                    const uint32_t to = start + slot * stage, bar = bar0 + 8 * slot, k = b * (kBlock / kElem);
                    if (p.drop != 1 + it || blockIdx.x != 0) copy_box<kCtas>(to, &map_x, k, m0, bar);
                    if (kCtas == 1) {
                        copy_box<kCtas>(to + kBytesA, &map_w, k, n0, bar);
                        copy_box<kCtas>(to + kBytesA + bytes_b / 2, &map_w, k, pairs ? p.outputs + n0 : n0 + g.n / 2, bar);
                    } else {
                        copy_box<kCtas>(to + kBytesA, &map_w, k, pair == 0 ? n0 : pairs ? p.outputs + n0 : n0 + g.n / 2, bar);
                    }
                }
            }
            /* copies already started land before the CTA exits (giving up does not stop them) */
            if (pair == 0)
                for (uint32_t j = it > g.stages ? it - g.stages : 0; j < it; ++j) {
                    const uint64_t w0 = gtimer();
                    while (!mbar_try(full + 8 * (j % g.stages), (j / g.stages) & 1u) && gtimer() - w0 < kWaitNs) {
                    }
                }
        }
        __syncwarp();
    } else if (warp == kEpilogueWarps + 1) {
        if (lane == 0 && pair == 0) {
            const uint32_t idesc = instr_desc<kFp8>(kCtas * kRowsA, g.n);
            uint32_t it = 0, seq = 0;
            bool ok = true;
            for (uint32_t tile = worker; ok && tile < tiles; tile += workers, ++seq) {
                const uint32_t acc = seq & 1u;
                if (seq >= 2 && !wait_bar(sums_empty + 8 * acc, ((seq >> 1) - 1) & 1u, abort)) break;
                tc_fence_after();
                const uint32_t d = tmem + acc * second;
                for (uint32_t b = b0; b < b1; ++b, ++it) {
                    const uint32_t slot = it % g.stages;
                    if (!wait_bar(full + 8 * slot, (it / g.stages) & 1u, abort)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a = start + slot * stage;
#pragma unroll
                    for (uint32_t k = 0; k < kBlock / 32; ++k)
                        mma<kCtas, kFp8>(d, smem_desc(a + k * 32), smem_desc(a + kBytesA + k * 32), idesc, b != b0 || k != 0);
                    commit<kCtas>(empty + 8 * slot);
                }
                if (ok) commit<kCtas>(sums_full + 8 * acc);
            }
            /* every MMA has ended, and its arrivals are here, before TMEM and this memory are given back */
            commit<kCtas>(drain);
        }
        if (lane == 0) {
            const uint64_t w0 = gtimer();
            while (!mbar_try(drain, 0) && gtimer() - w0 < 2 * kWaitNs) {
            }
        }
        __syncwarp();
    } else {
        const uint32_t quarter = warp & 3, half = warp >> 2; /* TMEM lanes, and every other 16 columns */
        const int64_t out_size = p.out_type == kBF16 ? 2 : 4, res_size = p.residual_type == kBF16 ? 2 : 4;
        const bool wide_out = ((reinterpret_cast<uintptr_t>(p.out) | (uintptr_t)(p.out_row * out_size)) & 15) == 0;
        const bool wide_res = ((reinterpret_cast<uintptr_t>(p.residual) | (uintptr_t)(p.residual_row * res_size)) & 15) == 0;
        uint32_t seq = 0;
        bool ok = true;
        for (uint32_t tile = worker; tile < tiles; tile += workers, ++seq) {
            const uint32_t acc = seq & 1u;
            const uint32_t n0 = tile / g.tiles_m * g.outs;
            Row r;
            r.token = (tile % g.tiles_m * kCtas + pair) * kRowsA + quarter * 32 + lane;
            r.scale = kFp8 && r.token < p.tokens ? __ldcg(p.x_scales + r.token) : 0.0f;
            if (kFp8 || p.bias != nullptr) {
                /* the accumulator's columns were last read two tiles ago, behind a barrier of the tile between */
                for (uint32_t c = tid; c < g.n; c += kEpilogueWarps * 32) {
                    const uint32_t n = c < g.outs ? n0 + c : n0 + c - g.outs;
                    const uint32_t row = c < g.outs ? n : p.outputs + n;
                    const bool have = n < p.outputs;
                    s->scale[acc][c] = kFp8 && have ? __ldcg(p.weight_scales + row) : 0.0f;
                    s->bias[acc][c] = p.bias != nullptr && have ? load1(p.bias, row, p.bias_type) : 0.0f;
                }
                epilogue_sync();
            }
            ok = ok && wait_bar(sums_full + 8 * acc, (seq >> 1) & 1u, abort);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            const uint32_t from = tmem + acc * second + ((quarter * 32) << 16);
            const float nan = __int_as_float(0x7fc00000);
            if (kCtas == 1 && g.split > 1) {
                /* the sums as [4 columns][token] in the stages, whose copies and MMAs have ended */
                if (!ok) s->failed = 1;
                for (uint32_t c = half * 16; ok && c < g.n; c += 32) {
                    float v[16];
                    tc_ld16(from + c, v);
                    tc_wait();
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<float4 *>(base + ((c / 4 + i) * kRowsA + quarter * 32 + lane) * 16) =
                            make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                }
                break; /* one tile; the rest below, with the cluster */
            }
            for (uint32_t c = half * 16; c < g.outs; c += 32) {
                float v[16], up[16];
                __syncwarp();
                if (ok) {
                    tc_ld16(from + c, v);
                    if (pairs) tc_ld16(from + g.outs + c, up);
                    tc_wait();
                }
                if (!ok) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = up[i] = nan;
                }
                r.n = n0 + c;
                if (r.token < p.tokens && r.n < p.outputs)
                    finish16(p, r, v, up, s->scale[acc] + c, s->bias[acc] + c, g.outs, wide_out, wide_res);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(kCtas == 2 ? map_rank(sums_empty + 8 * acc, 0) : sums_empty + 8 * acc);
        }
        __syncwarp();
    }
    if (kCtas == 1 && g.split > 1) {
        cluster_sync();
        if (warp < kEpilogueWarps && worker < tiles) {
            const int64_t out_size = p.out_type == kBF16 ? 2 : 4, res_size = p.residual_type == kBF16 ? 2 : 4;
            const bool wide_out = ((reinterpret_cast<uintptr_t>(p.out) | (uintptr_t)(p.out_row * out_size)) & 15) == 0;
            const bool wide_res = ((reinterpret_cast<uintptr_t>(p.residual) | (uintptr_t)(p.residual_row * res_size)) & 15) == 0;
            uint32_t bad = 0;
            for (uint32_t q = 0; q < g.split; ++q) bad |= load_cluster(map_rank(smem_u32(&s->failed), q));
            const uint32_t n0 = worker / g.tiles_m * g.outs, m = warp % 4 * 32 + lane;
            Row r;
            r.token = worker % g.tiles_m * kRowsA + m;
            r.scale = kFp8 && r.token < p.tokens ? __ldcg(p.x_scales + r.token) : 0.0f;
            /* 16 columns at a time, the cluster's CTAs and the two halves of a CTA's warps in turn */
            for (uint32_t c = (rank * 2 + warp / 4) * 16; c < g.outs; c += g.split * 32) {
                float v[16], up[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = up[i] = 0.0f;
                if (r.token < p.tokens)
                    for (uint32_t q = 0; q < g.split; ++q) {
                        const uint32_t from = map_rank(start, q);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float4 e = load_cluster4(from + ((c / 4 + i) * kRowsA + m) * 16);
                            v[4 * i] += e.x, v[4 * i + 1] += e.y, v[4 * i + 2] += e.z, v[4 * i + 3] += e.w;
                            if (pairs) {
                                const float4 u = load_cluster4(from + (((g.outs + c) / 4 + i) * kRowsA + m) * 16);
                                up[4 * i] += u.x, up[4 * i + 1] += u.y, up[4 * i + 2] += u.z, up[4 * i + 3] += u.w;
                            }
                        }
                    }
                if (bad) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = up[i] = __int_as_float(0x7fc00000);
                }
                r.n = n0 + c;
                if (r.token < p.tokens && r.n < p.outputs)
                    finish16(p, r, v, up, s->scale[0] + c, s->bias[0] + c, g.outs, wide_out, wide_res);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (kCtas == 2 || g.split > 1) cluster_sync(); /* nobody reads this CTA's memory any more */
    if (warp == 0) {
        if constexpr (kCtas == 1)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(g.columns) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(g.columns) : "memory");
    }
}

using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                            const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                            CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

cudaError_t encoder(Encode &f) {
    static std::atomic<void *> found{nullptr};
    void *at = found.load(std::memory_order_relaxed);
    if (at == nullptr) {
        cudaDriverEntryPointQueryResult result;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &at, 12000, cudaEnableDefault, &result);
        if (e != cudaSuccess) return e;
        if (result != cudaDriverEntryPointSuccess || at == nullptr) return cudaErrorNotSupported;
        found.store(at, std::memory_order_relaxed);
    }
    f = reinterpret_cast<Encode>(at);
    return cudaSuccess;
}

/* rows x inputs of 16-byte aligned rows, in boxes of 128 bytes of `box` rows; past its ends it reads zeros */
cudaError_t encode(CUtensorMap &map, const LinearParams &p, const void *at, int64_t row, uint64_t rows, uint32_t box) {
    Encode f;
    const cudaError_t e = encoder(f);
    if (e != cudaSuccess) return e;
    const uint32_t elem = p.type == kE4M3 ? 1 : 2;
    const cuuint64_t dims[2] = {p.inputs, rows};
    const cuuint64_t strides[1] = {rows == 1 ? ((uint64_t)p.inputs * elem + 15) / 16 * 16 : (uint64_t)row * elem};
    const cuuint32_t boxes[2] = {kBlock / elem, box}, steps[2] = {1, 1};
    const CUresult r = f(&map, p.type == kE4M3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                         const_cast<void *>(at), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

constexpr size_t kSmemLimit = 232448; /* 227 KB a CTA */

/* What is left to a launch once n, split and the number of CTAs to a tile are chosen. */
LinearShape shape_of(const LinearParams &p, uint32_t ctas, uint32_t n, uint32_t split) {
    LinearShape g;
    g.n = n;
    g.outs = p.activation == kSwiglu ? n / 2 : n;
    g.split = split;
    const uint32_t stage = kBytesA + n / ctas * kBlock;
    const uint32_t room = (uint32_t)(kSmemLimit - 1024 - sizeof(SharedTail)) / stage;
    g.stages = room < kMaxStages ? room : kMaxStages;
    g.rows_a = ctas == 2 || p.tokens >= kRowsA ? kRowsA : (p.tokens + 7) / 8 * 8;
    g.tiles_m = (p.tokens + ctas * kRowsA - 1) / (ctas * kRowsA);
    g.tiles_n = (p.outputs + g.outs - 1) / g.outs;
    g.blocks = (uint32_t)(((uint64_t)p.inputs * (p.type == kE4M3 ? 1 : 2) + kBlock - 1) / kBlock);
    g.columns = 32;
    while (g.columns < 2 * n) g.columns *= 2;
    return g;
}

template <int kCtas, bool kFp8>
cudaError_t launch_shape(const LinearParams &p, const LinearShape &g, int sms, cudaStream_t stream) {
    CUtensorMap map_x, map_w;
    cudaError_t e = encode(map_x, p, p.x, p.x_row, p.tokens, g.rows_a);
    if (e == cudaSuccess) e = encode(map_w, p, p.weight, p.weight_row, (uint64_t)p.outputs * (p.activation == kSwiglu ? 2 : 1), g.n / 2);
    if (e != cudaSuccess) return e;
    const size_t smem = 1024 + (size_t)g.stages * (kBytesA + g.n / kCtas * kBlock) + sizeof(SharedTail);
    e = cudaFuncSetAttribute(linear_kernel<kCtas, kFp8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemLimit);
    if (e != cudaSuccess) return e;
    const uint32_t tiles = g.tiles_m * g.tiles_n, group = kCtas * g.split;
    uint32_t workers = (uint32_t)sms / group;
    if (g.split > 1 || workers > tiles) workers = tiles;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(workers * group);
    cfg.blockDim = dim3(kLinearThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = group;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = group > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, linear_kernel<kCtas, kFp8>, p, map_x, map_w, g);
}

}  // namespace

cudaError_t launch_linear_as(const LinearParams &p, uint32_t ctas, uint32_t n, uint32_t split, int sms, cudaStream_t stream) {
    const LinearShape g = shape_of(p, ctas, n, split);
    if (p.type == kE4M3)
        return ctas == 2 ? launch_shape<2, true>(p, g, sms, stream) : launch_shape<1, true>(p, g, sms, stream);
    return ctas == 2 ? launch_shape<2, false>(p, g, sms, stream) : launch_shape<1, false>(p, g, sms, stream);
}

cudaError_t launch_linear(const LinearParams &p, int sms, cudaStream_t stream) {
    const uint64_t blocks = ((uint64_t)p.inputs * (p.type == kE4M3 ? 1 : 2) + kBlock - 1) / kBlock;
    const uint32_t rows = p.outputs * (p.activation == kSwiglu ? 2 : 1);
    uint32_t n = 256, split = 1;
    const uint32_t tiles_m = (p.tokens + kRowsA - 1) / kRowsA;
    while (n > 32 && (uint64_t)tiles_m * ((rows + n - 1) / n) < (uint64_t)sms) n /= 2;
    while (n <= 128 && split < 8 && 2 * (uint64_t)tiles_m * ((rows + n - 1) / n) * split <= (uint64_t)sms && split * 2 * 4 <= blocks) split *= 2;
    return launch_linear_as(p, p.tokens > 512 && n == 256 ? 2 : 1, n, split, sms, stream);
}

cudaError_t linear_status(int *status) {
    cudaError_t e = cudaMemcpyFromSymbol(status, g_linear_status, sizeof(int));
    const int zero = 0;
    if (e == cudaSuccess && *status != 0) e = cudaMemcpyToSymbol(g_linear_status, &zero, sizeof(int));
    return e;
}

}  // namespace ops
}  // namespace gdn
