/* gdn_linear.cu -- y = act(sx sw x W^T + bias) + residual on the tcgen05
 * tensor cores, for more tokens than gdn_linear_few.cu takes.
 *
 * D [tokens][rows of W] is cut into tiles of 128 tokens by up to 256 rows, or,
 * with two CTAs to a tile (cta_group::2), of 256 tokens: each of the two then
 * loads 128 tokens and half of the rows of W, which is what lets L2 keep up with
 * the tensor cores. BF16 operands go to kind::f16 and 8-bit ones to
 * kind::f8f6f4; both come as blocks of 128 bytes of k in the 128-byte swizzle,
 * so that the two differ in the instruction alone. For swiglu a tile holds the
 * same outputs of both halves of W side by side.
 *
 * The tensor cores cut the sums in TMEM to FP32 after each step of k, always
 * towards zero: over 352 steps (5632 inputs of BF16) results were 4.4e-6 off in the
 * 2-norm, where FP32 arithmetic is 5e-7. So TMEM takes a part of k at a time, and the
 * warps that empty it add these sums in registers, with rounding to nearest.
 *
 * A CTA has one warp that starts the TMA copies into a ring of stages, one
 * that starts the MMAs, and eight that add up the sums and take them to memory
 * (scales, bias, activation, residual) while the next MMAs run: there are two
 * accumulators. CTAs walk over the tiles, tokens first.
 *
 * Where there are too few tiles for all SMs, the CTAs of a cluster divide k:
 * each one's sums go to its shared memory, and each adds up, in the order of
 * the cluster's ranks, a part of the columns from all of them.
 *
 * Every wait is bounded (2 s). A CTA whose wait ran out writes NaN to its
 * outputs and sets g_linear_status.
 *
 * Measured. 4096 tokens of 2048 by 2 x 5632 of 8 bits with swiglu 65 to 75 us (2.5 to 2.9
 * PFLOP/s), of 5632 by 2048 of BF16 68 to 73 us (1.3 to 1.4 PFLOP/s), with an FP32 residual
 * and FP32 outputs 78 to 88: bound by the tensor cores (66 to 78 % of cycles) and, of
 * runs of a second, by the power limit (81, 79 and 95 to 101 us at 1.46 GHz); 128 tiles of
 * 256 by 256 for 74 pairs of CTAs leave 14 % of them idle. 64 tokens by 32000 of
 * BF16 25 us (5.2 TB/s), FP32 out 27 to 29, by 2 x 5632 with swiglu 13.6 us (3.5 TB/s):
 * bound by reading W, after which the last sums' way takes about 4 us: through
 * TMEM and the cluster, to memory, and the end of all CTAs. It begins 2.4 us after
 * the kernel before has ended, when the first blocks come.
 */
#include "gdn_linear.h"

#include <cuda.h>

#include <atomic>
#include <type_traits>

namespace gdn {
namespace ops {

namespace {

constexpr uint64_t kWaitNs = 2000000000ull;
constexpr uint32_t kEpilogueWarps = 8;
constexpr uint32_t kLinearThreads = (kEpilogueWarps + 4) * 32; /* three warpgroups: the last has two warps of use */
/* Registers a thread: 384 threads are launched with 168 (64512 in all); the warps with
 * the sums then take 216 and the others 64 (63488). With 168 the sums spilled. */
constexpr int kEpilogueRegs = 216, kOtherRegs = 64;
constexpr uint32_t kSplitRegs = kEpilogueWarps * 32 * kEpilogueRegs + 4 * 32 * kOtherRegs;
static_assert(kSplitRegs <= 168 * kLinearThreads, "more than the launch has: the split would wait for good");
constexpr uint32_t kBlock = 128;                  /* bytes of k in a row of a copy */
constexpr uint32_t kRowsA = 128;                  /* tokens of a CTA */
constexpr uint32_t kBytesA = kRowsA * kBlock;
constexpr uint32_t kMaxStages = 8;
constexpr uint32_t kMaxN = 256;
/* Blocks of k that TMEM adds up before the sums go on in registers. FP32 results of BF16 are off by 2.3e-7, 3.4e-7, 4.7e-7
 * and 7.0e-7 in the 2-norm with parts of 4, 6, 8 and 12 blocks, whatever the number of inputs, while FP32 arithmetic loses
 * more of longer sums (x.float() @ w.float().T 2.5e-7 of 1024 inputs, 3.9e-7 of 2048, 7.5e-7 of 5632): so parts grow with
 * the sum, and results stay under 2^-21 up to 2560 inputs. 2048 tokens of 1024 by 2048 take the same 12.7 us with 4 as with
 * 12, 64 of 2048 by 32000 27.3 with 6 and 27.2 with 12, 4096 of 2048 by 2048 39.5 and 36.3, 4096 of 5632 by 2048 91
 * and 85. The two sums of swiglu are off the same way, towards zero, which adds up: 4.6e-7 with 4 and 6.7e-7 with 6 (FP32
 * arithmetic 6.0e-7 of 2048 inputs, 1.2e-6 of 5632). BF16 results, which are rounded to 1.7e-3, and 8-bit operands, whose
 * products are short (3.0e-7 after 32 blocks, where FP32 arithmetic is 1.1e-6 off): 32. Even, for stages of two blocks. */
uint32_t chunk_of(const LinearParams &p, uint32_t blocks) {
    if (p.out_type == kBF16 || p.type == kE4M3) return 32;
    const bool pairs = p.activation == kSwiglu;
    const uint32_t most = pairs ? 6 : 12, chunk = (blocks / 8 + (pairs ? 0 : 2)) & ~1u;
    return chunk < 4 ? 4 : chunk < most ? chunk : most;
}

/* set when a wait of a kernel ran out; read and cleared by the host */
__device__ int g_linear_status;

/* a launch's tiles */
struct LinearShape {
    uint32_t n;        /* columns of a tile (rows of W): a multiple of 32 */
    uint32_t outs;     /* outputs of a tile: n, or n / 2 for swiglu */
    uint32_t split;    /* CTAs that divide k (one CTA to a tile), or 1 */
    uint32_t chunk;    /* blocks of k added up in TMEM */
    uint32_t sub;      /* 128-byte blocks of k in a stage: 1 or 2 */
    uint32_t stages;
    uint32_t rows_a;   /* rows of a copy of x: 128, or fewer where there are fewer tokens */
    uint32_t tiles_m, tiles_n, blocks; /* blocks: of k */
    uint32_t columns;  /* of TMEM */
};

struct SharedTail {
    uint64_t full[kMaxStages], empty[kMaxStages], sums_full[2], sums_empty[2], drain;
    uint32_t tmem, abort, failed;
    alignas(16) float scale[2][kMaxN], bias[2][kMaxN]; /* of a tile's columns */
};
constexpr uint32_t kTurnBytes = 32 * 64; /* of a warp: 32 tokens of 16 FP32 */

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
/* At a barrier of any CTA of the cluster, after tc_wait and tc_fence_before: what is handed over are columns of TMEM that
 * have been read. Relaxed, for no writes go with it: a release waited for the results on their way to memory, 1100
 * cycles (512 tokens of 2048 by 2048 9.0 us instead of 9.5). */
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
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
/* one lane of a converged warp */
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r != 0;
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
__device__ __forceinline__ float4 load_shared4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float load_shared(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint4 load_shared_u4(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void store_shared4(uint32_t addr, const uint4 &v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
/* a lane's row of 16 FP32 to its warp's buffer, for all lanes */
__device__ __forceinline__ void turn_rows(uint32_t to, uint32_t x, const float (&v)[16]) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i)
        store_shared4(to + ((i * 16) ^ x), make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]),
                                                      __float_as_uint(v[4 * i + 3])));
    __syncwarp();
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
 * (46-47), layout 2 (61-63). The high word is the same for all. */
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t smem_desc(uint32_t addr) { return (addr >> 4) | (1u << 16); }
/* D FP32 (bits 4-5 = 1); A and B (7-9, 10-12): BF16 is 1 of kind::f16, E4M3 0 of kind::f8f6f4; N >> 3 at 17, M >> 4 at 24 */
template <bool kFp8>
__device__ __forceinline__ uint32_t instr_desc(uint32_t m, uint32_t n) {
    return (1u << 4) | (kFp8 ? 0u : (1u << 7) | (1u << 10)) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

template <int kCtas, bool kFp8>
__device__ __forceinline__ void mma(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
#define GDN_MMA(GROUP, KIND)                                                                                              \
    asm volatile("{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n" \
                 " tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], da, db, %3, p;\n}\n" ::"r"(d),                     \
                 "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(kDescHigh)                                     \
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

/* kN sums of one token to values: v the sums, up those of the second half of W for swiglu.
 * `scale` and `bias` are those of the tile's columns from v's first on, with the second half's
 * `outs` further. */
template <int kN>
__device__ __forceinline__ void load_columns(const float *from, float (&v)[kN]) {
#pragma unroll
    for (int i = 0; i < kN; i += 4) {
        const float4 e = *reinterpret_cast<const float4 *>(from + i);
        v[i] = e.x, v[i + 1] = e.y, v[i + 2] = e.z, v[i + 3] = e.w;
    }
}
template <bool kFp8, bool pairs, int kN>
__device__ __forceinline__ void finish(const LinearParams &p, float row_scale, float (&v)[kN], float (&up)[kN], const float *scale,
                                       const float *bias, uint32_t outs) {
    if (kFp8) {
        float f[kN];
        load_columns(scale, f);
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] *= row_scale * f[i];
        if (pairs) {
            load_columns(scale + outs, f);
#pragma unroll
            for (int i = 0; i < kN; ++i) up[i] *= row_scale * f[i];
        }
    }
    if (p.bias != nullptr) {
        float f[kN];
        load_columns(bias, f);
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] += f[i];
        if (pairs) {
            load_columns(bias + outs, f);
#pragma unroll
            for (int i = 0; i < kN; ++i) up[i] += f[i];
        }
    }
    if (pairs || p.activation == kSilu) {
#pragma unroll
        for (int i = 0; i < kN; i += 2) split(silu2<true>(pair_of(v[i], v[i + 1])), v[i], v[i + 1]);
    } else if (p.activation == kGelu) {
#pragma unroll
        for (int i = 0; i < kN; i += 2) split(gelu2(pair_of(v[i], v[i + 1])), v[i], v[i + 1]);
    }
    if (pairs) {
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] *= up[i];
    }
}
__device__ __forceinline__ float4 load4(const void *p, int64_t i, int type) {
    if (type == kF32) return __ldcg(reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i));
    const uint2 w = __ldcg(reinterpret_cast<const uint2 *>(static_cast<const __nv_bfloat16 *>(p) + i));
    return make_float4(low_bf16(w.x), high_bf16(w.x), low_bf16(w.y), high_bf16(w.y));
}
/* four values as they are in memory */
__device__ __forceinline__ float4 value4(const uint4 &w, int type) {
    if (type == kF32) return make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w));
    return make_float4(low_bf16(w.x), high_bf16(w.x), low_bf16(w.y), high_bf16(w.y));
}
__device__ __forceinline__ void put4(void *p, int64_t i, int type, const float4 &v) {
    if (type == kF32)
        *reinterpret_cast<float4 *>(static_cast<float *>(p) + i) = v;
    else
        *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(p) + i) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}
/* Outputs n .. n + 3 of a token: their residuals (zeros without), and the rounding and the store. kWide: whole and
 * aligned, or past the end. */
template <bool kWide>
__device__ __forceinline__ float4 residual4(const LinearParams &p, uint32_t token, uint32_t n) {
    if (p.residual == nullptr || n >= p.outputs) return make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int64_t from = token * p.residual_row + n;
    if constexpr (kWide) {
        return load4(p.residual, from, p.residual_type);
    } else {
        float r[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < p.outputs) r[i] = load1(p.residual, from + i, p.residual_type);
        return make_float4(r[0], r[1], r[2], r[3]);
    }
}
template <bool kWide>
__device__ __forceinline__ void store4(const LinearParams &p, uint32_t token, uint32_t n, const float4 &v) {
    if (n >= p.outputs) return;
    const int64_t to = token * p.out_row + n;
    if (kWide) {
        put4(p.out, to, p.out_type, v);
        return;
    }
    const float value[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n + i < p.outputs) store1(p.out, to + i, p.out_type, value[i]);
}

/* 16 values of a lane of a block of 32 tokens by 16 outputs: those of output lane % 16 of every other token from lane / 16
 * on. `at`: the first one's place; `row`: from a token to the next; `left`: tokens from the first one on. */
template <typename T>
__device__ __forceinline__ void load_column(const T *at, int64_t row, uint32_t left, bool all, uint32_t (&v)[16]) {
    auto one = [](const T *from) {
        if constexpr (sizeof(T) == 4)
            return __ldcg(reinterpret_cast<const uint32_t *>(from));
        else
            return (uint32_t)__ldcg(reinterpret_cast<const unsigned short *>(from));
    };
    if (all) {
#pragma unroll
        for (int i = 0; i < 16; ++i, at += 2 * row) v[i] = one(at);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i, at += 2 * row) v[i] = 2u * i < left ? one(at) : 0u;
    }
}
template <typename T>
__device__ __forceinline__ void store_column(T *at, int64_t row, uint32_t left, bool all, const float (&v)[16]) {
    if (all) {
#pragma unroll
        for (int i = 0; i < 16; ++i, at += 2 * row) store1(at, v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i, at += 2 * row)
            if (2u * i < left) store1(at, v[i]);
    }
}

/* The outputs of a tile from the sums of the kSplit CTAs of its cluster, in the order of their ranks: four of a token at
 * a time, in turn over the cluster's threads. The loads of several fours go out together, those of the residual too: 300
 * tokens of 5632 by 2048 with a residual took 19.8 us with one four at a time and 18.2 so. */
template <bool kFp8, bool pairs, bool kWide, int kSplit>
__device__ __forceinline__ void join_parts(const LinearParams &p, const LinearShape &g, const SharedTail &s, uint32_t start, uint32_t rank,
                                           uint32_t worker, uint32_t tid) {
    constexpr int kEach = 8 / kSplit, kHalves = pairs ? 2 : 1;
    constexpr uint32_t kStep = kSplit * kEpilogueWarps * 32;
    uint32_t bad = 0, from[kSplit];
#pragma unroll
    for (uint32_t q = 0; q < kSplit; ++q) {
        from[q] = map_rank(start, q);
        bad |= load_cluster(map_rank(smem_u32(&s.failed), q));
    }
    const uint32_t n0 = worker / g.tiles_m * g.outs, m0 = worker % g.tiles_m * kRowsA, pieces = g.outs / 4;
    const uint32_t items = min(kRowsA, p.tokens - m0) * pieces;
    for (uint32_t first = rank * kEpilogueWarps * 32 + tid; first < items; first += kEach * kStep) {
        float4 e[kEach][kHalves][kSplit];
        float4 r[kEach];
        float row_scale[kEach];
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const uint32_t i = min(first + k * kStep, items - 1), m = i / pieces, q4 = i % pieces; /* past the end: read, and not used */
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
#pragma unroll
                for (int q = 0; q < kSplit; ++q) e[k][h][q] = load_cluster4(from[q] + m * g.n * 4 + (((q4 + h * pieces) ^ (m & 7)) * 16));
            r[k] = residual4<kWide>(p, m0 + m, n0 + q4 * 4);
            row_scale[k] = kFp8 ? __ldcg(p.x_scales + m0 + m) : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const uint32_t i = first + k * kStep, m = i / pieces, q4 = i % pieces;
            if (i >= items) break;
            float v[kHalves][4];
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                v[h][0] = v[h][1] = v[h][2] = v[h][3] = 0.0f;
#pragma unroll
                for (int q = 0; q < kSplit; ++q)
                    v[h][0] += e[k][h][q].x, v[h][1] += e[k][h][q].y, v[h][2] += e[k][h][q].z, v[h][3] += e[k][h][q].w;
            }
            if (bad) v[0][0] = v[0][1] = v[0][2] = v[0][3] = __int_as_float(0x7fc00000);
            finish<kFp8, pairs>(p, row_scale[k], v[0], v[kHalves - 1], s.scale[0] + q4 * 4, s.bias[0] + q4 * 4, g.outs);
            store4<kWide>(p, m0 + m, n0 + q4 * 4, make_float4(v[0][0] + r[k].x, v[0][1] + r[k].y, v[0][2] + r[k].z, v[0][3] + r[k].w));
        }
    }
}

/* How a block of results goes to memory: in pieces of four values, where rows of out and of the residual are whole
 * aligned ones, or value by value, without a residual and with one. Compiled apart: together they spilled 2.9 KB a
 * thread. */
enum Way { kPieces = 0, kValues = 1, kValuesAdded = 2 };

template <int kCtas, bool kFp8, bool pairs, int kWay>
__global__ void __launch_bounds__(kLinearThreads, 1)
    linear_kernel(const __grid_constant__ LinearParams p, const __grid_constant__ CUtensorMap map_x,
                  const __grid_constant__ CUtensorMap map_w, const LinearShape g) {
    extern __shared__ uint8_t raw[];
    constexpr bool kWide = kWay == kPieces;
    constexpr uint32_t kElem = kFp8 ? 1 : 2;
    const uint32_t start = (smem_u32(raw) + 1023u) & ~1023u;
    uint8_t *base = raw + (start - smem_u32(raw));
    const uint32_t bytes_b = g.n / kCtas * kBlock, block = kBytesA + bytes_b, stage = g.sub * block;
    uint8_t *turn_buffers = base + g.stages * stage;
    SharedTail *s = reinterpret_cast<SharedTail *>(turn_buffers + kEpilogueWarps * kTurnBytes);
    volatile uint32_t *abort = &s->abort;
    const uint32_t full = smem_u32(s->full), empty = smem_u32(s->empty), sums_full = smem_u32(s->sums_full),
                   sums_empty = smem_u32(s->sums_empty), drain = smem_u32(&s->drain);
    /* taken from one lane, so that the compiler sees that all lanes of a warp go the same way */
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t rank = kCtas == 1 && g.split == 1 ? 0 : cluster_rank(), pair = kCtas == 2 ? rank : 0;
    const uint32_t group = kCtas * g.split, worker = blockIdx.x / group, workers = gridDim.x / group;
    const uint32_t tiles = g.tiles_m * g.tiles_n;
    const uint32_t b0 = kCtas == 1 ? (uint32_t)((uint64_t)g.blocks * rank / g.split) : 0;
    const uint32_t b1 = kCtas == 1 ? (uint32_t)((uint64_t)g.blocks * (rank + 1) / g.split) : g.blocks;

    if (warp == kEpilogueWarps) {
        if (lane == 0) {
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
        __syncwarp();
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
    if (kCtas == 2) {
        __syncthreads();
        cluster_sync(); /* the other CTA's barriers are ready */
    } else if (warp == kEpilogueWarps) {
        /* the copies need the barriers, which this warp has made, and not TMEM */
        asm volatile("bar.arrive 2, %0;" ::"n"(kLinearThreads) : "memory");
    } else {
        asm volatile("bar.sync 2, %0;" ::"n"(kLinearThreads) : "memory");
    }
    tc_fence_after();
    wait_for_previous();
    let_next_start();
    const uint32_t second = g.columns / 2; /* columns from one accumulator to the other */

    if (warp >= kEpilogueWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        /* Whole warps walk and wait, and one lane of them acts: the instructions of the tensor cores take
         * uniform registers. Slots and phases are counted, not divided for: with the loops of a single
         * lane that divided, a stage took 1000 cycles whatever its size. */
        if (warp == kEpilogueWarps) {
            const uint32_t bar0 = kCtas == 2 ? map_rank(full, 0) : full; /* the pair's MMAs wait at the first CTA's */
            const uint32_t bytes = kCtas * (g.rows_a * kBlock + bytes_b);
            const uint32_t dropped = blockIdx.x == 0 ? p.drop : 0;
            uint32_t slot = 0, phase = 1, it = 0, made = 0; /* phase: of the slot's last use, whose end is waited for */
            bool ok = true;
            for (uint32_t tile = worker; ok && tile < tiles; tile += workers) {
                const uint32_t m0 = (tile % g.tiles_m * kCtas + pair) * kRowsA, n0 = tile / g.tiles_m * g.outs;
                const uint32_t n1 = pairs ? p.outputs + n0 : n0 + g.n / 2;
                for (uint32_t b = b0; b < b1; b += g.sub, ++it) {
                    /* a new barrier's wait for the phase before its first returns at once */
                    ok = __all_sync(0xffffffffu, wait_bar(empty + 8 * slot, phase, abort));
                    if (!ok) break;
                    const uint32_t here = min(g.sub, b1 - b), bar = bar0 + 8 * slot;
                    if (elect_one()) {
                        if (pair == 0) mbar_expect_tx(full + 8 * slot, here * bytes);
                        for (uint32_t i = 0; i < here; ++i) {
                            const uint32_t to = start + slot * stage + i * block, k = (b + i) * (kBlock / kElem);
                            if (dropped != made + i + 1) copy_box<kCtas>(to, &map_x, k, m0, bar);
                            if (kCtas == 2) {
                                copy_box<kCtas>(to + kBytesA, &map_w, k, pair == 0 ? n0 : n1, bar);
                            } else {
                                copy_box<kCtas>(to + kBytesA, &map_w, k, n0, bar);
                                if (pairs) copy_box<kCtas>(to + kBytesA + bytes_b / 2, &map_w, k, n1, bar);
                            }
                        }
                    }
                    __syncwarp();
                    made += here;
                    if (++slot == g.stages) slot = 0, phase ^= 1;
                }
            }
            /* copies already started land before the CTA exits (giving up does not stop them) */
            if (pair == 0 && lane == 0)
                for (uint32_t j = it > g.stages ? it - g.stages : 0; j < it; ++j) {
                    const uint64_t w0 = gtimer();
                    while (!mbar_try(full + 8 * (j % g.stages), (j / g.stages) & 1u) && gtimer() - w0 < kWaitNs) {
                    }
                }
        }
        if (warp == kEpilogueWarps + 1 && pair == 0) {
            const uint32_t idesc = instr_desc<kFp8>(kCtas * kRowsA, g.n), tmem = s->tmem;
            uint32_t slot = 0, phase = 0, acc = 0, acc_phase = 1;
            bool ok = true;
            for (uint32_t tile = worker; ok && tile < tiles; tile += workers) {
                for (uint32_t c0 = b0; ok && c0 < b1; c0 += g.chunk) {
                    const uint32_t c1 = min(c0 + g.chunk, b1), d = tmem + acc * second;
                    ok = __all_sync(0xffffffffu, wait_bar(sums_empty + 8 * acc, acc_phase, abort));
                    if (!ok) break;
                    tc_fence_after();
                    for (uint32_t b = c0; b < c1; b += g.sub) {
                        ok = __all_sync(0xffffffffu, wait_bar(full + 8 * slot, phase, abort));
                        if (!ok) break;
                        tc_fence_after();
                        if (elect_one()) {
                            const uint32_t a = smem_desc(start + slot * stage), w = smem_desc(start + slot * stage + kBytesA);
#pragma unroll
                            for (uint32_t k = 0; k < kBlock / 32; ++k) mma<kCtas, kFp8>(d, a + 2 * k, w + 2 * k, idesc, b != c0 || k != 0);
                            if (g.sub == 2 && b + 1 < c1) {
#pragma unroll
                                for (uint32_t k = 0; k < kBlock / 32; ++k)
                                    mma<kCtas, kFp8>(d, a + (block >> 4) + 2 * k, w + (block >> 4) + 2 * k, idesc, true);
                            }
                            commit<kCtas>(empty + 8 * slot);
                            if (b + g.sub >= c1) commit<kCtas>(sums_full + 8 * acc);
                        }
                        __syncwarp();
                        if (++slot == g.stages) slot = 0, phase ^= 1;
                    }
                    acc_phase ^= acc;
                    acc ^= 1;
                }
            }
            /* every MMA has ended, and its arrivals are here, before TMEM and this memory are given back */
            if (elect_one()) commit<kCtas>(drain);
            __syncwarp();
        }
        if (warp == kEpilogueWarps + 1 && lane == 0) {
            const uint64_t w0 = gtimer();
            while (!mbar_try(drain, 0) && gtimer() - w0 < 2 * kWaitNs) {
            }
        }
        __syncwarp();
        if (kCtas == 1 && g.split > 1) cluster_sync(); /* with the sums */
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpilogueRegs));
        const uint32_t quarter = warp & 3, half = warp >> 2; /* TMEM lanes, and every other 16 columns */
        const uint32_t tmem = s->tmem;
        const bool has_res = kWide ? p.residual != nullptr : kWay == kValuesAdded, f32_out = p.out_type == kF32;
        const bool out16 = ((reinterpret_cast<uintptr_t>(p.out) | (uintptr_t)p.out_row * 2 | (uintptr_t)p.outputs * 2) & 15) == 0; /* BF16 */
        /* 16-byte piece q of row r of a warp's buffer at r * 64 + (q ^ (r / 2 % 4)) * 16 */
        const uint32_t turn_base = smem_u32(turn_buffers) + warp * kTurnBytes;
        const uint32_t turn_out = turn_base + lane * 64, turn_out_x = (lane >> 1 & 3) * 16;
        const uint32_t turn_in = turn_base + (lane >> 2) * 64 + (((lane & 3) ^ (lane >> 3 & 3)) * 16);
        uint32_t seq = 0, turn = 0;
        bool ok = true;
        for (uint32_t tile = worker; tile < tiles; tile += workers, ++turn) {
            const uint32_t n0 = tile / g.tiles_m * g.outs;
            const uint32_t row0 = (tile % g.tiles_m * kCtas + pair) * kRowsA + quarter * 32, token = row0 + lane;
            const float row_scale = kFp8 && token < p.tokens ? __ldcg(p.x_scales + token) : 0.0f;
            if (has_res && token < p.tokens) {
                /* this row's part of the residual on its way to L2, in pieces of 128 bytes, while the MMAs run */
                const int64_t size = p.residual_type == kF32 ? 4 : 2;
                const char *row = static_cast<const char *>(p.residual) + (token * p.residual_row + n0) * size;
                const uint32_t bytes = (uint32_t)size * min(g.outs, p.outputs - n0);
                for (uint32_t i = half * 128; i < bytes; i += 256) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + i));
            }
            float *scale = s->scale[turn & 1], *bias = s->bias[turn & 1];
            if (kFp8 || p.bias != nullptr) {
                /* these were last read two tiles ago, behind a barrier of the tile between */
                for (uint32_t c = tid; c < g.n; c += kEpilogueWarps * 32) {
                    const uint32_t n = c < g.outs ? n0 + c : n0 + c - g.outs;
                    const uint32_t row = c < g.outs ? n : p.outputs + n;
                    const bool have = n < p.outputs;
                    scale[c] = kFp8 && have ? __ldcg(p.weight_scales + row) : 0.0f;
                    bias[c] = p.bias != nullptr && have ? load1(p.bias, row, p.bias_type) : 0.0f;
                }
                epilogue_sync();
            }
            /* This thread's sums: 16 columns a set. The tile's outputs are units of 16, in turn the first and the
             * second half's of the warps; for swiglu the sets 2 j and 2 j + 1 are one unit of either half of W. */
            constexpr int kSets = kMaxN / 32;
            float sum[kSets][16];
            auto unit = [&](int set) { return (uint32_t)(pairs ? set / 2 : set) * 2 + half; };
            auto have = [&](int set) { return unit(set) * 16 < g.outs; };
            auto column = [&](int set) { return unit(set) * 16 + (pairs && (set & 1) ? g.outs : 0); };
            const bool rows = row0 < p.tokens; /* this warp has any */
            /* The residual of the sets, two ahead of the one that is finished, the first two from before the last sums
             * are there: pieces of four values of eight tokens apart, or (not kWide) a column of every other token. */
            constexpr int kStep = pairs ? 2 : 1;
            const uint32_t piece = (lane & 3) * 4, column16 = lane & 15, high = kWide ? lane >> 2 : lane >> 4;
            const uint32_t left = row0 + high < p.tokens ? p.tokens - row0 - high : 0; /* tokens from this lane's first one on */
            const int64_t out_at = (row0 + high) * p.out_row + n0 + (kWide ? 0 : column16);
            const int64_t res_at = (row0 + high) * p.residual_row + n0 + (kWide ? piece : column16);
            const bool all = row0 + 32 <= p.tokens;
            uint4 e[kWide ? 2 : 1][4];
            uint32_t f[kWay == kValuesAdded ? 2 : 1][16];
            auto load_residual = [&](int set) {
                const int to = set / kStep & 1;
                const uint32_t c = unit(set) * 16;
                if (!has_res || set >= kSets || !have(set)) return;
                if constexpr (kWide) {
                    /* past the ends, where nothing is stored, the last token's and the tile's first outputs: the loads are not
                     * branched around, so that nothing waits for one of them */
                    const uint32_t n = n0 + c + piece < p.outputs ? n0 + c + piece : n0;
                    int64_t at[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) at[i] = min(row0 + high + 8 * i, p.tokens - 1) * p.residual_row + n;
                    if (p.residual_type == kF32) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) e[to][i] = __ldcg(reinterpret_cast<const uint4 *>(static_cast<const float *>(p.residual) + at[i]));
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint2 w = __ldcg(reinterpret_cast<const uint2 *>(static_cast<const __nv_bfloat16 *>(p.residual) + at[i]));
                            e[to][i].x = w.x, e[to][i].y = w.y;
                        }
                    }
                } else if constexpr (kWay == kValuesAdded) {
                    if (n0 + c + column16 < p.outputs) {
                        if (p.residual_type == kF32)
                            load_column(static_cast<const float *>(p.residual) + res_at + c, p.residual_row, left, all, f[to]);
                        else
                            load_column(static_cast<const __nv_bfloat16 *>(p.residual) + res_at + c, p.residual_row, left, all, f[to]);
                    }
                }
            };
            for (uint32_t b = b0; b < b1; b += g.chunk, ++seq) {
                const uint32_t acc = seq & 1u;
                if (b + g.chunk >= b1 && !(kCtas == 1 && g.split > 1)) {
                    load_residual(0);
                    load_residual(kStep);
                }
                ok = ok && wait_bar(sums_full + 8 * acc, (seq >> 1) & 1u, abort);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t from = tmem + acc * second + ((quarter * 32) << 16);
                /* In place of columns that the tile does not have its first ones are loaded: around branches the compiler moves
                 * each load's values to other registers, and so waits for one load after the other (64 tokens of 2048
                 * by 2048 7.8 us, 7.2 so). */
                if (!rows) {
                } else if (b == b0) {
#pragma unroll
                    for (int set = 0; set < kSets; ++set) tc_ld16(from + (have(set) ? column(set) : 0), sum[set]);
                    tc_wait();
                } else {
#pragma unroll
                    for (int set = 0; set < kSets; set += 2) {
                        if (!have(set)) break;
                        float v[2][16];
#pragma unroll
                        for (int j = 0; j < 2; ++j) tc_ld16(from + (have(set + j) ? column(set + j) : 0), v[j]);
                        tc_wait();
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int i = 0; i < 16; ++i) sum[set + j][i] += v[j][i];
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(kCtas == 2 ? map_rank(sums_empty + 8 * acc, 0) : sums_empty + 8 * acc);
            }
            if (!ok) {
#pragma unroll
                for (int set = 0; set < kSets; ++set)
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum[set][i] = __int_as_float(0x7fc00000);
            }
            if (kCtas == 1 && g.split > 1) {
                /* to the stages, whose copies and MMAs have ended: piece q of a token at q ^ (token % 8) */
                if (!ok) s->failed = 1;
#pragma unroll
                for (int set = 0; set < kSets; ++set)
                    if (ok && rows && have(set)) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            *reinterpret_cast<float4 *>(base + (quarter * 32 + lane) * g.n * 4 + (((column(set) / 4 + i) ^ (lane & 7)) * 16)) =
                                make_float4(sum[set][4 * i], sum[set][4 * i + 1], sum[set][4 * i + 2], sum[set][4 * i + 3]);
                    }
                break; /* one tile; the rest below, with the cluster */
            }
            /* A row of 16 values a lane is turned so that four lanes have one: whole sectors of memory are read and
             * written. One lane's pieces are eight rows apart. */
            if (!rows) {
            } else if (kWide && !has_res && !f32_out && out16) {
                /* BF16: two units to a turn, four pieces of eight values a row */
#pragma unroll
                for (int set = 0; set < kSets; set += 2 * kStep) {
                    if (!have(set)) break;
                    const uint32_t c = unit(set) * 16, c2 = c + 32; /* of the second unit */
                    const bool second_one = c2 < g.outs;
                    finish<kFp8, pairs>(p, row_scale, sum[set], sum[set + (pairs ? 1 : 0)], scale + c, bias + c, g.outs);
                    if (second_one)
                        finish<kFp8, pairs>(p, row_scale, sum[set + kStep], sum[set + kStep + (pairs ? 1 : 0)], scale + c2, bias + c2, g.outs);
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float(&v)[16] = sum[set + (i >> 1) * kStep];
                        const int o = (i & 1) * 8;
                        store_shared4(turn_out + ((i * 16) ^ turn_out_x),
                                      make_uint4(pack_bf16(v[o], v[o + 1]), pack_bf16(v[o + 2], v[o + 3]), pack_bf16(v[o + 4], v[o + 5]),
                                                 pack_bf16(v[o + 6], v[o + 7])));
                    }
                    __syncwarp();
                    const uint32_t n = ((lane & 2) ? c2 : c) + (lane & 1) * 8;
                    __nv_bfloat16 *to = static_cast<__nv_bfloat16 *>(p.out) + out_at + n;
                    if (n < g.outs && n0 + n < p.outputs) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (8u * i < left) *reinterpret_cast<uint4 *>(to + i * 8 * p.out_row) = load_shared_u4(turn_in + i * 512);
                    }
                }
            } else if (kWide) {
#pragma unroll
                for (int set = 0; set < kSets; set += kStep) {
                    const uint32_t c = unit(set) * 16;
                    if (!have(set) || n0 + c >= p.outputs) break;
                    finish<kFp8, pairs>(p, row_scale, sum[set], sum[set + (pairs ? 1 : 0)], scale + c, bias + c, g.outs);
                    turn_rows(turn_out, turn_out_x, sum[set]);
                    float4 v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = load_shared4(turn_in + i * 512);
                    if (has_res) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float4 r = value4(e[set / kStep & 1][i], p.residual_type);
                            v[i].x += r.x, v[i].y += r.y, v[i].z += r.z, v[i].w += r.w;
                        }
                    }
                    const bool have_piece = n0 + c + piece < p.outputs;
                    const int64_t to = out_at + c + piece;
                    if (f32_out) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (have_piece && 8u * i < left) put4(p.out, to + i * 8 * p.out_row, kF32, v[i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (have_piece && 8u * i < left) put4(p.out, to + i * 8 * p.out_row, kBF16, v[i]);
                    }
                    load_residual(set + 2 * kStep);
                }
            } else {
#pragma unroll
                for (int set = 0; set < kSets; set += kStep) {
                    const uint32_t c = unit(set) * 16;
                    if (!have(set) || n0 + c >= p.outputs) break;
                    float v[16];
                    finish<kFp8, pairs>(p, row_scale, sum[set], sum[set + (pairs ? 1 : 0)], scale + c, bias + c, g.outs);
                    turn_rows(turn_out, turn_out_x, sum[set]);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        v[i] = load_shared(turn_base + (2 * i + high) * 64 + (((column16 >> 2) ^ (i & 3)) << 4) + (column16 & 3) * 4);
                        if constexpr (kWay == kValuesAdded)
                            v[i] += __uint_as_float(p.residual_type == kF32 ? f[set / kStep & 1][i] : f[set / kStep & 1][i] << 16);
                    }
                    if (n0 + c + column16 < p.outputs) {
                        if (f32_out)
                            store_column(static_cast<float *>(p.out) + out_at + c, p.out_row, left, all, v);
                        else
                            store_column(static_cast<__nv_bfloat16 *>(p.out) + out_at + c, p.out_row, left, all, v);
                    }
                    load_residual(set + 2 * kStep);
                }
            }
        }
        __syncwarp();
        if (kCtas == 1 && g.split > 1) {
            cluster_sync();
            if (worker < tiles) {
                if (g.split == 2)
                    join_parts<kFp8, pairs, kWide, 2>(p, g, *s, start, rank, worker, tid);
                else if (g.split == 4)
                    join_parts<kFp8, pairs, kWide, 4>(p, g, *s, start, rank, worker, tid);
                else
                    join_parts<kFp8, pairs, kWide, 8>(p, g, *s, start, rank, worker, tid);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (kCtas == 2 || g.split > 1) cluster_sync(); /* nobody reads this CTA's memory any more */
    if (warp == 0) {
        const uint32_t tmem = s->tmem;
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

constexpr uint32_t kSmemRest = 1024 + kEpilogueWarps * kTurnBytes + sizeof(SharedTail);

/* 128-byte blocks of k */
uint32_t blocks_of(const LinearParams &p) { return (uint32_t)(((uint64_t)p.inputs * (p.type == kE4M3 ? 1 : 2) + kBlock - 1) / kBlock); }

/* What is left to a launch once n, split and the number of CTAs to a tile are chosen. */
LinearShape shape_of(const LinearParams &p, uint32_t ctas, uint32_t n, uint32_t split, uint32_t sub) {
    LinearShape g;
    g.n = n;
    g.outs = p.activation == kSwiglu ? n / 2 : n;
    g.split = split;
    g.sub = sub;
    const uint32_t stage = sub * (kBytesA + n / ctas * kBlock);
    const uint32_t room = (uint32_t)(kSmemLimit - kSmemRest) / stage;
    g.stages = room < kMaxStages ? room : kMaxStages;
    g.rows_a = ctas == 2 || p.tokens >= kRowsA ? kRowsA : (p.tokens + 7) / 8 * 8;
    g.tiles_m = (p.tokens + ctas * kRowsA - 1) / (ctas * kRowsA);
    g.tiles_n = (p.outputs + g.outs - 1) / g.outs;
    g.blocks = blocks_of(p);
    g.chunk = chunk_of(p, g.blocks);
    g.columns = 32;
    while (g.columns < 2 * n) g.columns *= 2;
    return g;
}

template <int kCtas, bool kFp8, bool pairs, int kWay>
cudaError_t launch_shape(const LinearParams &p, const LinearShape &g, int sms, cudaStream_t stream) {
    CUtensorMap map_x, map_w;
    cudaError_t e = encode(map_x, p, p.x, p.x_row, p.tokens, g.rows_a);
    if (e == cudaSuccess) e = encode(map_w, p, p.weight, p.weight_row, (uint64_t)p.outputs * (pairs ? 2 : 1), kCtas == 2 || pairs ? g.n / 2 : g.n);
    if (e != cudaSuccess) return e;
    const size_t smem = kSmemRest + (size_t)g.stages * g.sub * (kBytesA + g.n / kCtas * kBlock);
    e = cudaFuncSetAttribute(linear_kernel<kCtas, kFp8, pairs, kWay>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemLimit);
    if (e != cudaSuccess) return e;
    static const cudaError_t registers = [] {
        cudaFuncAttributes attr;
        const cudaError_t error = cudaFuncGetAttributes(&attr, linear_kernel<kCtas, kFp8, pairs, kWay>);
        return error != cudaSuccess ? error : (uint32_t)attr.numRegs * kLinearThreads < kSplitRegs ? cudaErrorInvalidKernelImage : cudaSuccess;
    }();
    if (registers != cudaSuccess) return registers;
    const uint32_t tiles = g.tiles_m * g.tiles_n, group = kCtas * g.split;
    uint32_t workers = (uint32_t)sms / group;
    if (g.split > 1 || workers > tiles) workers = tiles;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(workers * group);
    cfg.blockDim = dim3(kLinearThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; /* as launch_overlapped */
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = group;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = group > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, linear_kernel<kCtas, kFp8, pairs, kWay>, p, map_x, map_w, g);
}

/* whether all results, and their residuals, are pieces of four values on their boundaries */
bool whole_pieces(const LinearParams &p) {
    auto aligned = [&](const void *at, int64_t row, int type) {
        const uintptr_t size = type == kF32 ? 4 : 2;
        return ((reinterpret_cast<uintptr_t>(at) | (p.tokens == 1 ? 0 : (uintptr_t)row * size)) & (4 * size - 1)) == 0;
    };
    return p.outputs % 4 == 0 && aligned(p.out, p.out_row, p.out_type) &&
           (p.residual == nullptr || aligned(p.residual, p.residual_row, p.residual_type));
}

uint64_t tiles_of(const LinearParams &p, uint32_t ctas, uint32_t n) {
    const uint32_t outs = p.activation == kSwiglu ? n / 2 : n;
    return (uint64_t)((p.tokens + ctas * kRowsA - 1) / (ctas * kRowsA)) * ((p.outputs + outs - 1) / outs);
}
/* What a call may take: n a multiple of 32, so that the eight pieces of a row of sums that tokens take in turn are the row's own;
 * two CTAs where there are tokens for both; a divided k of at least four blocks a CTA, with tiles whose clusters run at once
 * (of clusters of four and eight not as many CTAs as there are SMs: 13 of eight did, 16 did not). */
bool possible(const LinearParams &p, uint32_t ctas, uint32_t n, uint32_t split, int sms) {
    if (n == 0 || n > kMaxN || n % 32 != 0 || ctas == 0 || ctas > (p.tokens > kRowsA ? 2u : 1u)) return false;
    if (split == 1) return true;
    const uint64_t most = (uint64_t)sms * (split < 4 ? 8 : split == 4 ? 7 : 6) / 8;
    return ctas == 1 && (split == 2 || split == 4 || split == 8) && tiles_of(p, 1, n) * split <= most && blocks_of(p) / split >= 4;
}

cudaError_t launch_linear_as(const LinearParams &p, uint32_t ctas, uint32_t n, uint32_t split, int sms, cudaStream_t stream) {
    if (!possible(p, ctas, n, split, sms)) return cudaErrorInvalidValue;
    const uint32_t sub = n <= 128 ? 2 : 1; /* stages of 36 to 64 KB: three at least */
    const LinearShape g = shape_of(p, ctas, n, split, sub);
    auto pick = [&](auto pairs, auto way) {
        constexpr bool kPairs = decltype(pairs)::value;
        constexpr int kWay = decltype(way)::value;
        if (p.type == kE4M3) return ctas == 2 ? launch_shape<2, true, kPairs, kWay> : launch_shape<1, true, kPairs, kWay>;
        return ctas == 2 ? launch_shape<2, false, kPairs, kWay> : launch_shape<1, false, kPairs, kWay>;
    };
    auto pick_way = [&](auto pairs, bool wide) {
        if (wide) return pick(pairs, std::integral_constant<int, kPieces>());
        return p.residual == nullptr ? pick(pairs, std::integral_constant<int, kValues>()) : pick(pairs, std::integral_constant<int, kValuesAdded>());
    };
    const bool wide = whole_pieces(p);
    auto *launch = p.activation == kSwiglu ? pick_way(std::true_type(), wide) : pick_way(std::false_type(), wide);
    return launch(p, g, sms, stream);
}

}  // namespace

/* The tiles of a call are those for which this estimate is least. What it knows, in us on 148 SMs: a block of k takes
 * 0.00144 n + 0.05 in one CTA and 0.00128 n + 0.024 in two, of which each computes half the columns of both; a launch
 * 4.5 or 5.2; each tile of a CTA 1.0; the last tile's results, where they go value by value, 0.01 n; a cluster that
 * divides k 0.9 + 0.04 a CTA. Against all tiles of 138 calls (17 to 4096 tokens, 128 to 5632 inputs, 501 to 32000
 * outputs, both types, all activations; gdn_b200_test_linear_tiles) its choices were 1.0 % slower than the best tiles in the mean, 6 %
 * or more for a tenth of them and 25 % at most; 256 columns undivided are 85 % slower in the mean and up to five times. */
cudaError_t launch_linear(const LinearParams &p, int sms, cudaStream_t stream) {
    if (p.tiles != 0) return launch_linear_as(p, p.tiles & 15, p.tiles >> 4 & 4095, p.tiles >> 16, sms, stream);
    const uint32_t blocks = blocks_of(p);
    float least = 3.4e38f;
    uint32_t ctas = 1, n = 256, split = 1;
    const bool whole = whole_pieces(p);
    for (uint32_t c = 1; c <= (p.tokens > kRowsA ? 2u : 1u); ++c)
        for (uint32_t width = 32; width <= kMaxN; width += 32) {
            const uint64_t tiles = tiles_of(p, c, width);
            const float block = c == 2 ? 0.00128f * width + 0.024f : 0.00144f * width + 0.053f;
            for (uint32_t s = 1; s <= 8 && possible(p, c, width, s, sms); s *= 2) {
                const uint64_t waves = (tiles * c * s + sms - 1) / sms;
                const float t = (float)waves * ((float)((blocks + s - 1) / s) * block + 1.0f) + (c == 2 ? 5.2f : 4.5f) +
                                (whole ? 0.0f : 0.01f * width) + (s > 1 ? 0.9f + 0.04f * s : 0.0f);
                if (t < least) least = t, ctas = c, n = width, split = s;
            }
        }
    return launch_linear_as(p, ctas, n, split, sms, stream);
}

cudaError_t linear_status(int *status) {
    cudaError_t e = cudaMemcpyFromSymbol(status, g_linear_status, sizeof(int));
    const int zero = 0;
    if (e == cudaSuccess && *status != 0) e = cudaMemcpyToSymbol(g_linear_status, &zero, sizeof(int));
    return e;
}

}  // namespace ops
}  // namespace gdn
