/* gdn_delta_chunk.cu -- the gated delta rule over prompts, 64 tokens at a
 * time on the tensor cores (BF16 q, k, v; FP32 states in the pool).
 *
 * Within a chunk of C = 64 tokens, with G_i the sum of the log decays up to
 * token i and khat, qhat the (normalised) keys and queries:
 *   A_ij = beta_i e^(G_i - G_j) khat_i.khat_j (j < i),   T = (I + A)^-1
 *   P_ij = scale e^(G_i - G_j) qhat_i.khat_j (j <= i)
 *   R = beta (V - e^G khat S0^T),   D = T R
 *   O = scale e^G qhat S0^T + (P T) R
 *   S = e^(G_C) S0 + sum_j e^(G_C - G_j) D_j khat_j^T
 * T and P T do not depend on the state, so a first kernel forms them for all
 * chunks at once; a second one walks each sequence's chunks. The columns of
 * S0^T (value rows) do not mix: a CTA takes VB of them through the whole
 * sequence, with the state in registers.
 *
 * The state has to come out as FP32 arithmetic would give it, from BF16
 * tensor cores with FP32 accumulators: k and q enter as they are (exact), their
 * norms and the decays scale rows of results, and each FP32 operand enters
 * as three BF16 terms that sum to it (24 bits): S0, R, D, T and P T. The terms
 * of an operand are columns of one MMA (N = 3 VB), whose sums are added when they
 * are read back. (With two terms for T the states' errors against 64 bits were
 * up to 7e-7 for independent keys and 5e-6 where all keys of a sequence are
 * alike; with two for P T the outputs were 2.4e-6 off before their rounding to
 * BF16, which then went the other way for one in a thousand.)
 *
 * A token whose k, v, g or beta is not finite makes NaN of its own output and
 * of all that follow, as the rule does, but must not reach the tokens before it
 * through the zeros of T and P T above their diagonals (0 NaN). So its row of R
 * enters the MMA as zeros (and its row of A as the identity's); its row of D
 * is then set to NaN, with which the state follows, and so are the outputs of
 * the chunk from it on.
 *
 * What bounds the walk is the chain of one chunk: three rounds of MMAs, each
 * waiting for the epilogue of the one before. Measured with 8 heads of 256 x
 * 256: 4096 tokens 171 us (2500 token by token), of which the first kernel
 * takes 27 and a chunk of the second 4100 cycles; 24 prompts of up to 2047
 * tokens 626 us.
 */
#include "gdn_ops.h"

#include <cuda_bf16.h>

namespace gdn {
namespace ops {

namespace {

constexpr int kC = 64;      /* tokens of a chunk */
constexpr uint64_t kWaitNs = 2000000000ull;

/* per (chunk, value head): three BF16 terms of [T; P T] in the MMA's layout,
 * then four rows of 64 floats and the chunk's decay */
constexpr uint32_t kTermBytes = 2 * kC * 128;       /* 128 rows of 64 BF16 */
constexpr uint32_t kPairBytes = 3 * kTermBytes;
constexpr uint32_t kScalBytes = (4 * kC + 4) * 4;
constexpr uint32_t kRecordBytes = (kPairBytes + kScalBytes + 127) & ~127u;
enum { kScalC = 0, kScalBeta = 1, kScalQ = 2, kScalEnd = 3, kScalDecay = 4 };

/* set when a wait of a kernel ran out; read and cleared by the host */
__device__ int g_chunk_status;

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
/* One arrival for the warp, after all its lanes got here: a barrier's arrivals
 * are served one after the other, and 256 of them took longer than the MMAs
 * they were to start. */
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
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
/* Bounded wait; false when the CTA gives up (here or elsewhere). The clock and
 * the other warps' word are looked at now and then: they cost issue slots that
 * the epilogues need. kPause: nobody waits for this warp to wake at once. */
template <bool kPause = false>
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile uint32_t *abort) {
    if (mbar_try(bar, parity)) return true;
    const uint64_t t0 = gtimer();
    while (true) {
        if (kPause) __nanosleep(100);
#pragma unroll 1
        for (int i = 0; i < 16; ++i)
            if (mbar_try(bar, parity)) return true;
        if (*abort) return false;
        if (gtimer() - t0 > kWaitNs) {
            *abort = 1;
            atomicExch(&g_chunk_status, 1);
            return false;
        }
    }
}
/* the same for a whole warp, with one answer */
template <bool kPause = false>
__device__ __forceinline__ bool wait_bar_warp(uint32_t bar, uint32_t parity, volatile uint32_t *abort) {
    return __all_sync(0xffffffffu, wait_bar<kPause>(bar, parity, abort));
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

/* Shared-memory matrix descriptors in the 128-byte swizzle (rows of 128 bytes,
 * 16-byte piece p of row r at p ^ (r & 7), 1 KB per eight rows): start >> 4
 * (bits 0-13), leading offset >> 4 (16-29), stride offset >> 4 (32-45),
 * version 1 (46-47), layout 2 (61-63). The stride of 1 KB goes from one group
 * of eight rows to the next. K-major (a row is an index of M or N): the leading
 * offset is not used. MN-major (a row is an index of K, its 64 elements are
 * indexes of M or N): it goes to the next 64 of them. The high word is the
 * same for all; a later start only adds to the low word. */
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc(uint32_t addr, uint32_t lead) { return (addr >> 4) | ((lead >> 4) << 16); }
/* kind::f16: D FP32, A and B BF16, A and B K-major or MN-major */
__host__ __device__ constexpr uint32_t instr_desc(uint32_t m, uint32_t n, bool a_mn, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((n >> 3) << 17) |
           ((m >> 4) << 24);
}
/* D (+)= A B; a and b are low words of descriptors */
__device__ __forceinline__ void mma(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(kDescHigh)
        : "memory");
}
/* one lane of a converged warp */
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
/* eight FP32 columns of this thread's TMEM lane; tc_wait before the values are used */
__device__ __forceinline__ void tc_ld8(uint32_t addr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
}
__device__ __forceinline__ void tc_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr));
}
__device__ __forceinline__ void tc_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
/* pairs of FP32 values */
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t pack2(float lo, float hi) { return pack2(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ void unpack2(uint64_t v, float &lo, float &hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
/* y = f x + y and y = x + y */
__device__ __forceinline__ void scale_add(float f, const float (&x)[8], float (&y)[8]) {
    const uint64_t ff = pack2(f, f);
#pragma unroll
    for (int i = 0; i < 8; i += 2) unpack2(fma2(ff, pack2(x[i], x[i + 1]), pack2(y[i], y[i + 1])), y[i], y[i + 1]);
}
__device__ __forceinline__ void add_to(const float (&x)[8], float (&y)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) unpack2(add2(pack2(x[i], x[i + 1]), pack2(y[i], y[i + 1])), y[i], y[i + 1]);
}
/* whether all are finite: by a product with zeros, in three steps of packed operations */
__device__ __forceinline__ bool all_finite(const float (&x)[8]) {
    const uint64_t none = pack2(0.0f, 0.0f);
    const uint64_t a = fma2(pack2(x[0], x[1]), none, fma2(pack2(x[2], x[3]), none, none));
    const uint64_t b = fma2(pack2(x[4], x[5]), none, fma2(pack2(x[6], x[7]), none, none));
    float lo, hi;
    unpack2(add2(a, b), lo, hi);
    return lo + hi == 0.0f;
}
/* the sums of the three terms' columns (VB apart): eight value rows starting at addr */
template <int VB>
__device__ __forceinline__ void tc_sum3(uint32_t addr, float (&x)[8]) {
    uint32_t a[8], b[8], c[8];
    __syncwarp();
    tc_ld8(addr, a);
    tc_ld8(addr + VB, b);
    tc_ld8(addr + 2 * VB, c);
    tc_wait();
#pragma unroll
    for (int i = 0; i < 8; i += 2)
        unpack2(add2(pack2(a[i], a[i + 1]), add2(pack2(b[i], b[i + 1]), pack2(c[i], c[i + 1]))), x[i], x[i + 1]);
}

/* 16-byte piece `piece` of row `row` in the 128-byte swizzle */
__device__ __forceinline__ uint32_t piece_at(uint32_t row, uint32_t piece) { return row * 128u + ((piece ^ (row & 7u)) << 4); }

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
/* Eight values as three BF16 terms, eight significant bits each from the top:
 * with the 24 bits of FP32 their sum is the value itself (an infinity or a
 * NaN makes NaN terms, as it would make every sum it enters). Row `row` of an
 * MN-major operand: the eight-value pieces term * VB / 8 + sub, eight of them to
 * a row of 128 bytes, the further ones from piece kAt on in a second block
 * (`second` bytes on). */
template <int VB, uint32_t kAt = 0>
__device__ __forceinline__ void put_terms(uint8_t *base, uint32_t second, uint32_t row, uint32_t sub, const float (&x)[8]) {
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(x[i]);
#pragma unroll
    for (int term = 0; term < 3; ++term) {
        const uint32_t piece = term * (VB / 8) + sub;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __byte_perm(r[2 * i], r[2 * i + 1], 0x7632);
        uint8_t *to = piece < 8 ? base + piece_at(row, piece) : base + second + piece_at(row, (piece & 7) + kAt);
        *reinterpret_cast<uint4 *>(to) = make_uint4(w[0], w[1], w[2], w[3]);
        if (term < 2) {
            /* minus the term: a mixed FMA takes it from the pair, on the pipe
             * that the packing leaves free (masks and packed subtractions took
             * 220 cycles a call, 2 warps to a scheduler) */
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float lo = __uint_as_float(r[2 * i]), hi = __uint_as_float(r[2 * i + 1]);
                asm("{\n .reg .b16 l, h, m;\n mov.b32 {l, h}, %2;\n mov.b16 m, 0xbf80;\n"
                    " fma.rn.f32.bf16 %0, l, m, %0;\n fma.rn.f32.bf16 %1, h, m, %1;\n}"
                    : "+f"(lo), "+f"(hi)
                    : "r"(w[i]));
                r[2 * i] = __float_as_uint(lo);
                r[2 * i + 1] = __float_as_uint(hi);
            }
        }
    }
}

/* `rows` tokens from t0 on of one head (zeros up to 64) as the rows `first`
 * .. first + 63 of blocks of 64 columns (`block` bytes apart) in the 128-byte
 * swizzle */
template <int K, uint32_t kThreads>
__device__ __forceinline__ void load_rows(uint32_t tile, uint32_t block, uint32_t first, const __nv_bfloat16 *x, int64_t t0,
                                          int64_t stride, uint32_t rows, uint32_t thread) {
    /* a thread keeps its piece of a row and goes down in steps of a multiple
     * of eight rows, so that its place in the swizzle stays the same */
    constexpr uint32_t kPieces = K / 8, kWide = kPieces < kThreads / 8 ? kPieces : kThreads / 8, kStep = kThreads / kWide;
    static_assert(kStep % 8 == 0 && kPieces % kWide == 0 && kC % kStep == 0, "loader shape");
    const uint32_t r0 = thread / kWide;
#pragma unroll
    for (uint32_t c0 = 0; c0 < kPieces; c0 += kWide) {
        const uint32_t c = c0 + thread % kWide;
        uint32_t dst = tile + (c >> 3) * block + piece_at(first + r0, c & 7);
        const __nv_bfloat16 *src = x + (t0 + r0) * stride + c * 8;
#pragma unroll
        for (uint32_t r = 0; r < kC; r += kStep) {
            const bool there = r0 + r < rows;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(there ? src : x), "r"(there ? 16u : 0u)
                         : "memory");
            dst += kStep * 128;
            src += kStep * stride;
        }
    }
}
__device__ __forceinline__ void cp_async_wait_all() {
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

/* Records are numbered so that no prefix sum over the sequences is needed:
 * chunk c of sequence n has number starts[n] / 64 + n + c. */
__host__ __device__ __forceinline__ uint32_t record_of(uint32_t t0, uint32_t n) { return t0 / kC + n; }

/* Programmatic dependent launch: the second kernel may set up while the first
 * one finishes, and waits for it before it reads anything of its. */
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

/* ------------------------------------------------------------ first kernel */

/* order[i]: the i-th longest sequence. The walks start in this order, so that
 * the last to start are short. The CTAs of the first value head take the
 * sequences in turn; a place is the number of sequences that come before. Each
 * looks at all of them: very many stay in their own order, whose walks are dealt
 * out over many rounds anyway (300000 single tokens of one small head: 460 ms in
 * order of length, 16 in their own). */
constexpr uint32_t kMaxOrdered = 4096;
__device__ __forceinline__ void place_sequences(const DeltaParams &p, uint32_t *order) {
    if (p.N > kMaxOrdered) {
        for (uint32_t n = blockIdx.x * blockDim.x + threadIdx.x; n < p.N; n += gridDim.x * blockDim.x) order[n] = n;
        return;
    }
    for (uint32_t n = blockIdx.x; n < p.N; n += gridDim.x) {
        uint32_t a, b, before = 0;
        sequence_tokens(p, n, a, b);
        const uint32_t len = b - a;
        for (uint32_t m = threadIdx.x; m < p.N; m += blockDim.x) {
            sequence_tokens(p, m, a, b);
            before += b - a > len || (b - a == len && m < n);
        }
        __shared__ uint32_t total;
        __syncthreads();
        if (threadIdx.x == 0) total = 0;
        __syncthreads();
        if (before) atomicAdd(&total, before);
        __syncthreads();
        if (threadIdx.x == 0) order[total] = n;
    }
}

/* Two threads per row of [K; Q] form, from the MMA's products, its row of A (k)
 * or of P (q). T = (I + A)^-1 by blocks,
 *   [[a 0] [c b]]^-1 = [[a^-1 0] [-b^-1 c a^-1, b^-1]],
 * the four of 16 on the diagonal by substitution, a warp each and a lane per
 * row; the products, and P T, with mma.sync of TF32 parts (x = x0 + x1 + x2, six
 * of the nine products: 24 bits of each; with x0 + x1 and three products, 21
 * bits, the states of like keys were 1.4e-6 off). What bounds it is the chain
 * of these steps, 15000 cycles alone and 22000 where three CTAs share an SM to
 * fill its gaps: 27 us for 64 chunks of 8 heads of 256. */
constexpr int kPrepThreads = 256;
constexpr uint32_t kLdA = kC + 8, kLdP = kC + 4; /* row strides of A, T and X, and of P: fragments without bank conflicts */

/* The FP32 matrices take the place of [K; Q] once the MMAs have read it. */
template <int K>
struct PrepSmem {
    static constexpr uint32_t kTile = 0;                                  /* [K; Q] */
    static constexpr uint32_t kA = 0;                                     /* A, then T */
    static constexpr uint32_t kP = kA + kC * kLdA * 4;
    static constexpr uint32_t kX = kP + kC * kLdP * 4;                    /* c a^-1 */
    static constexpr uint32_t kMat = kX + 32 * kLdA * 4;
    static constexpr uint32_t kG = (K / 64) * kTermBytes > kMat ? (K / 64) * kTermBytes : kMat;
    static constexpr uint32_t kRows = 7;                                  /* G hi, lo, beta, norms of k, q, two of decays */
    static constexpr uint32_t kBar = kG + kRows * kC * 4;
    static constexpr uint32_t kBytes = kBar + 32 + 1024;                  /* room to align */
};

/* Row `lane` of the inverse of a 16 x 16 unit lower triangular block, given
 * its part below the diagonal: x (I + A) = e, from the last column on; each x_j
 * that is final is taken off the columns before it. */
__device__ __forceinline__ void invert16(float *A, uint32_t lane) {
    uint64_t y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = pack2((uint32_t)(2 * j) == lane ? 1.0f : 0.0f, (uint32_t)(2 * j + 1) == lane ? 1.0f : 0.0f);
#pragma unroll
    for (int j = 15; j >= 1; --j) {
        float lo, hi;
        unpack2(y[j / 2], lo, hi);
        const float x = -((j & 1) ? hi : lo);
        const uint64_t xx = pack2(x, x);
        const ulonglong2 *row = reinterpret_cast<const ulonglong2 *>(A + j * kLdA);
#pragma unroll
        for (int l = 0; l < j; l += 4) {
            const ulonglong2 a = row[l / 4];
            if (l + 1 < j) y[l / 2] = fma2(xx, a.x, y[l / 2]);
            if (l + 3 < j) y[l / 2 + 1] = fma2(xx, a.y, y[l / 2 + 1]);
            if ((j & 1) && l + 4 > j) {
                /* the last column before an odd j: the pair's other half is x_j itself */
                float alo, ahi, ylo, yhi;
                unpack2(j - 1 == l ? a.x : a.y, alo, ahi);
                unpack2(y[j / 2], ylo, yhi);
                y[j / 2] = pack2(fmaf(x, alo, ylo), yhi);
            }
        }
    }
    __syncwarp();
    if (lane < 16) {
        ulonglong2 *out = reinterpret_cast<ulonglong2 *>(A + lane * kLdA);
#pragma unroll
        for (int j = 0; j < 8; j += 2) out[j / 2] = make_ulonglong2(y[j], y[j + 1]);
    }
}

/* Fragments of m16n8k8, g = lane / 4, t = lane % 4, each element in three TF32
 * parts, 11 significant bits each from the top: all 24 of FP32 */
constexpr int kParts = 3;
struct FragA {
    uint32_t v[kParts][4];
};
struct FragB {
    uint32_t v[kParts][2];
};
template <int N>
__device__ __forceinline__ void tf32_parts(float x, uint32_t (&v)[kParts][N], int i) {
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
        v[part][i] = __float_as_uint(x) & 0xFFFFE000u;
        x -= __uint_as_float(v[part][i]);
    }
}
/* rows r .. r + 15, columns c .. c + 7 of m */
__device__ __forceinline__ FragA frag_a(const float *m, uint32_t ld, uint32_t r, uint32_t c, uint32_t lane) {
    FragA f;
    const float *p = m + (r + (lane >> 2)) * ld + c + (lane & 3);
    tf32_parts(p[0], f.v, 0);
    tf32_parts(p[8 * ld], f.v, 1);
    tf32_parts(p[4], f.v, 2);
    tf32_parts(p[8 * ld + 4], f.v, 3);
    return f;
}
/* rows (k) r .. r + 7, columns (n) c .. c + 7 of m */
__device__ __forceinline__ FragB frag_b(const float *m, uint32_t ld, uint32_t r, uint32_t c, uint32_t lane) {
    FragB f;
    const float *p = m + (r + (lane & 3)) * ld + c + (lane >> 2);
    tf32_parts(p[0], f.v, 0);
    tf32_parts(p[4 * ld], f.v, 1);
    return f;
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
/* The products of at least 2^-22 of the first, by size in three accumulators:
 * they do not wait for one another, and small sums are not lost in large ones. */
__device__ __forceinline__ void mma_parts(float (&d)[3][4], const FragA &a, const FragB &b) {
    mma_tf32(d[0], a.v[2], b.v[0]);
    mma_tf32(d[1], a.v[1], b.v[0]);
    mma_tf32(d[2], a.v[0], b.v[0]);
    mma_tf32(d[0], a.v[0], b.v[2]);
    mma_tf32(d[1], a.v[0], b.v[1]);
    mma_tf32(d[0], a.v[1], b.v[1]);
}
__device__ __forceinline__ float parts_sum(const float (&d)[3][4], int e) { return d[2][e] + (d[0][e] + d[1][e]); }
/* rows r .. r + 15, columns c .. c + 7 of out = sign * a b, over kK columns of a;
 * rows of kLdA */
template <int kK>
__device__ __forceinline__ void product_tile(float *out, const float *a, const float *b, float sign, uint32_t r, uint32_t c,
                                             uint32_t lane) {
    float d[3][4] = {};
#pragma unroll
    for (int k = 0; k < kK; k += 8) mma_parts(d, frag_a(a, kLdA, r, k, lane), frag_b(b, kLdA, k, c, lane));
    float *p = out + (r + (lane >> 2)) * kLdA + c + 2 * (lane & 3);
    *reinterpret_cast<float2 *>(p) = make_float2(sign * parts_sum(d, 0), sign * parts_sum(d, 1));
    *reinterpret_cast<float2 *>(p + 8 * kLdA) = make_float2(sign * parts_sum(d, 2), sign * parts_sum(d, 3));
}
/* two neighbouring values of a row of the record as three BF16 terms */
__device__ __forceinline__ void put_pair3(uint8_t *rec, uint32_t row, uint32_t col, float x, float y) {
    uint8_t *p = rec + piece_at(row, col >> 3) + (col & 7) * 2;
#pragma unroll
    for (int term = 0; term < 3; ++term) {
        const uint32_t w = bf16_pair(x, y);
        *reinterpret_cast<uint32_t *>(p + term * kTermBytes) = w;
        x -= __uint_as_float(w << 16);
        y -= __uint_as_float(w & 0xFFFF0000u);
    }
}

__device__ __forceinline__ void load8(const float *p, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void store8(float *p, const float (&x)[8]) {
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
/* e^x for a decay: the product with log2 e rounds by 2^-24 |x|, and
 * |x| e^x stays below 0.37 */
__device__ __forceinline__ float decay_exp(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}

template <int K>
__global__ void __launch_bounds__(kPrepThreads, 3) chunk_prep_kernel(const __grid_constant__ DeltaParams p, uint8_t *records, uint32_t *order) {
    using L = PrepSmem<K>;
    extern __shared__ uint8_t raw[];
    uint8_t *sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    const uint32_t base = smem_u32(sm);
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rec = blockIdx.x, h = blockIdx.y, hq = h / (p.HV / p.H);
    __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(p.out);
    if (h == 0) place_sequences(p, order);

    /* the sequence whose records hold number rec: the last one whose first
     * record is at or before it. All threads look at once where that takes
     * fewer rounds than halving. N: the tokens after the last sequence. */
    uint32_t t0, t1, n;
    auto begins_by = [&](uint32_t m) {
        uint32_t a, b;
        if (m < p.N) {
            sequence_tokens(p, m, a, b);
        } else {
            sequence_tokens(p, p.N - 1, b, a);
        }
        return record_of(a, m) <= rec;
    };
    if (p.N <= 8 * kPrepThreads) {
        n = 0;
        for (uint32_t m = 1; m <= p.N; m += kPrepThreads)
            n += (uint32_t)__syncthreads_count(m + tid <= p.N && begins_by(m + tid));
    } else {
        uint32_t lo = 0, hi = p.N;
        while (lo < hi) {
            const uint32_t mid = (lo + hi + 1) / 2;
            if (begins_by(mid))
                lo = mid;
            else
                hi = mid - 1;
        }
        n = lo;
    }
    if (n == 0 && p.starts != nullptr) {
        /* tokens before the first sequence give zeros */
        sequence_tokens(p, 0, t0, t1);
        const uint32_t z1 = min(t0, (rec + 1) * kC);
        for (uint32_t t = rec * kC; t < z1; ++t)
            for (uint32_t i = tid; i < p.V; i += kPrepThreads)
                out[(int64_t)t * p.out_token + (int64_t)h * p.out_head + i] = __float2bfloat16_rn(0.0f);
        if (rec < record_of(t0, 0)) return;
    }
    if (n == p.N) {
        uint32_t a;
        sequence_tokens(p, p.N - 1, a, t0);
        t0 += (rec - record_of(t0, p.N)) * kC;
        for (uint32_t t = t0; t < min(p.tokens, t0 + kC); ++t)
            for (uint32_t i = tid; i < p.V; i += kPrepThreads)
                out[(int64_t)t * p.out_token + (int64_t)h * p.out_head + i] = __float2bfloat16_rn(0.0f);
        return;
    }
    sequence_tokens(p, n, t0, t1);
    const uint32_t chunk = rec - record_of(t0, n);
    t0 += chunk * kC;
    if (t0 >= t1) return;
    const uint32_t rows = min((uint32_t)kC, t1 - t0);
    uint8_t *record = records + ((size_t)rec * p.HV + h) * kRecordBytes;

    const __nv_bfloat16 *q = static_cast<const __nv_bfloat16 *>(p.q) + (int64_t)hq * p.q_head;
    const __nv_bfloat16 *k = static_cast<const __nv_bfloat16 *>(p.k) + (int64_t)hq * p.k_head;
    load_rows<K, kPrepThreads>(base + L::kTile, kTermBytes, 0, k, t0, p.k_token, rows, tid);
    load_rows<K, kPrepThreads>(base + L::kTile, kTermBytes, kC, q, t0, p.q_token, rows, tid);

    float *A = reinterpret_cast<float *>(sm + L::kA), *P = reinterpret_cast<float *>(sm + L::kP);
    float *X = reinterpret_cast<float *>(sm + L::kX), *G = reinterpret_cast<float *>(sm + L::kG);
    uint32_t *first_bad = reinterpret_cast<uint32_t *>(sm + L::kBar + 24); /* the first token whose row of A is not finite */
    float *Glo = G + kC, *bet = G + 2 * kC, *kin = G + 3 * kC, *qin = G + 4 * kC, *dec_i = G + 5 * kC, *dec_j = G + 6 * kC;
    const uint32_t bar = base + L::kBar;
    uint32_t *slot = reinterpret_cast<uint32_t *>(sm + L::kBar + 8);
    volatile uint32_t *abort = reinterpret_cast<volatile uint32_t *>(sm + L::kBar + 16);
    if (tid == 0) {
        mbar_init(bar, 1);
        *abort = 0;
        *first_bad = kC;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(128u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 1) {
        /* sums of the log decays in 64 bits, kept as two floats: differences of
         * nearby sums stay exact however far the sums have gone. e^-10000 is
         * 0 like any decay below it. */
        double s[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t r = 2 * lane + i;
            const float gv = r < rows ? p.g[(int64_t)(t0 + r) * p.g_token + (int64_t)h * p.g_head] : 0.0f;
            s[i] = (double)(gv < -10000.0f ? -10000.0f : gv);
            bet[r] = r < rows ? p.beta[(int64_t)(t0 + r) * p.beta_token + (int64_t)h * p.beta_head] : 0.0f;
        }
        s[1] += s[0];
        double run = s[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double below = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= (uint32_t)o) run += below;
        }
        double before = __shfl_up_sync(0xffffffffu, run, 1);
        if (lane == 0) before = 0.0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const double x = before + s[i];
            const float hi32 = (float)x;
            G[2 * lane + i] = hi32;
            Glo[2 * lane + i] = (float)(x - (double)hi32);
        }
    }
    cp_async_wait_all();
    fence_async();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    /* not before this CTA has its TMEM: a CTA of the second kernel that took
     * the rest would wait for this one for good */
    pdl_launch();
    if (warp == 0 && elect_one()) {
        /* [K; Q] [K; Q]^T: the first 64 columns are wanted, and the diagonal for the norms */
        const uint32_t at = desc(base + L::kTile, 16);
#pragma unroll
        for (int kk = 0; kk < K / 16; ++kk) {
            const uint32_t off = ((kk / 4) * kTermBytes + (kk % 4) * 32) >> 4;
            mma(tmem, at + off, at + off, instr_desc(2 * kC, 2 * kC, false, false), kk != 0);
        }
        commit(bar);
    }
    if (!wait_bar_warp(bar, 0, abort)) *first_bad = 0; /* nothing that could pass for a result */
    tc_fence_after();
    /* rows 32 (warp % 4) .. + 31 of [K; Q], one a lane: token i of k or of q */
    const uint32_t row = 32 * (warp & 3) + lane, lanes = (32 * (warp & 3)) << 16, i = row & (kC - 1);
    const bool is_p = row >= (uint32_t)kC, low = i >= 32; /* uniform in a warp */
    if (warp < 4) {
        /* its norm, from the diagonal */
        uint32_t r[32];
        float ss = 0.0f;
        __syncwarp();
        tc_ld32(tmem + lanes + 32 * warp, r);
        tc_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e)
            if ((int)lane == e) ss = __uint_as_float(r[e]);
        const float inv = p.normalize ? 1.0f / sqrtf(ss + 1e-6f) : 1.0f;
        if (is_p)
            qin[i] = inv * p.scale;
        else
            kin[i] = inv;
    }
    __syncthreads(); /* [K; Q] has been read: the matrices may take its place */
    /* the record's rows of scalars */
    if (warp < 2) {
        float *sc = reinterpret_cast<float *>(record + kPairBytes);
        const float eg = expf(G[i] + Glo[i]);
        const bool there = i < rows;
        sc[kScalC * kC + i] = there ? eg * kin[i] : 0.0f;
        sc[kScalBeta * kC + i] = bet[i];
        sc[kScalQ * kC + i] = eg * qin[i];
        sc[kScalEnd * kC + i] = there ? expf((G[kC - 1] - G[i]) + (Glo[kC - 1] - Glo[i])) * kin[i] : 0.0f;
        if (i == kC - 1) sc[kScalDecay * kC] = eg;
        /* the two factors of the decays between the halves of the chunk */
        if (i < 32)
            dec_j[i] = expf((G[32] - G[i]) + (Glo[32] - Glo[i])) * kin[i];
        else
            dec_i[i] = expf((G[i] - G[32]) + (Glo[i] - Glo[32]));
    }
    __syncthreads();
    /* row i of A or P: warps 0-3 columns 0 .. 31, warps 4-7 the others. e^(G_i -
     * G_j) of the lower left quarter is the product of e^(G_i - G_32) and
     * e^(G_32 - G_j), neither above 1 where nothing grows; the upper right one is
     * zero. */
    {
        const bool left = warp < 4;
        const uint32_t c0 = left ? 0 : 32;
        float *dst = (is_p ? P + i * kLdP : A + i * kLdA) + c0;
        uint32_t r[32];
        if (low || left) {
            __syncwarp();
            tc_ld32(tmem + lanes + c0, r);
            tc_wait();
        }
        float f = is_p ? qin[i] : bet[i] * kin[i], zero = 0.0f; /* zero: NaN when one of the row is not finite */
        if (low != left) {
            /* the quarter with the diagonal */
            const float gi = G[i], gl = Glo[i];
            const int last = (int)(i & 31) - (is_p ? 0 : 1); /* the last column with a product */
#pragma unroll
            for (int c = 0; c < 32; c += 8) {
                float gj[8], lj[8], kj[8], x[8];
                load8(G + c0 + c, gj);
                load8(Glo + c0 + c, lj);
                load8(kin + c0 + c, kj);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    /* for all columns: taken only where wanted, it cost a branch each (5200 cycles for the 32) */
                    const float y = f * kj[e] * decay_exp((gi - gj[e]) + (gl - lj[e])) * __uint_as_float(r[c + e]);
                    x[e] = c + e <= last ? y : 0.0f;
                    zero = fmaf(x[e], 0.0f, zero);
                }
                store8(dst + c, x);
            }
        } else {
            if (low) f *= dec_i[i];
#pragma unroll
            for (int c = 0; c < 32; c += 8) {
                float dj[8], x[8];
                load8(dec_j + c, dj);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = low ? f * dj[e] * __uint_as_float(r[c + e]) : 0.0f;
                    zero = fmaf(x[e], 0.0f, zero);
                }
                store8(dst + c, x);
            }
        }
        if (!is_p && !(zero == 0.0f)) atomicMin(first_bad, i);
    }
    tc_fence_before();
    __syncthreads();
    const uint32_t bad = *first_bad;
    if (bad < (uint32_t)kC) {
        /* rows that the tokens before do not need; the scalars make NaN of them */
        for (uint32_t x = tid; x < (kC - bad) * kC; x += kPrepThreads) {
            A[(bad + x / kC) * kLdA + x % kC] = 0.0f;
            P[(bad + x / kC) * kLdP + x % kC] = 0.0f;
        }
        if (warp < 2 && i >= bad) {
            float *sc = reinterpret_cast<float *>(record + kPairBytes);
            sc[kScalC * kC + i] = sc[kScalBeta * kC + i] = sc[kScalQ * kC + i] = __int_as_float(0x7fc00000);
        }
        __syncthreads();
    }
    constexpr uint32_t kDiag = kLdA + 1;
    if (warp < 4) invert16(A + 16 * warp * kDiag, lane);
    __syncthreads();
    /* blocks of 32: warps 0, 1 the first, 2, 3 the second, 8 columns each */
    float *B = A + 32 * (warp >> 1) * kDiag, *XB = X + 16 * (warp >> 1) * kLdA;
    if (warp < 4) product_tile<16>(XB, B + 16 * kLdA, B, 1.0f, 0, 8 * (warp & 1), lane);
    __syncthreads();
    if (warp < 4) product_tile<16>(B + 16 * kLdA, B + 16 * kDiag, XB, -1.0f, 0, 8 * (warp & 1), lane);
    __syncthreads();
    product_tile<32>(X, A + 32 * kLdA, A, 1.0f, 16 * (warp >> 2), 8 * (warp & 3), lane);
    __syncthreads();
    product_tile<32>(A + 32 * kLdA, A + 32 * kDiag, X, -1.0f, 16 * (warp >> 2), 8 * (warp & 3), lane);
    __syncthreads();
    /* the record: T in the rows of the chunk's k, P T in those of its q (both
     * lower triangular); the two change places from chunk to chunk */
    const uint32_t t_row = (chunk & 1) ? kC : 0, p_row = kC - t_row;
    for (uint32_t x = tid; x < kC * 8; x += kPrepThreads) {
        const uint32_t r = x >> 3, c = (x & 7) * 8;
        float v[8];
        load8(A + r * kLdA + c, v);
        uint32_t w[3][4];
#pragma unroll
        for (int term = 0; term < 3; ++term)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[term][e] = bf16_pair(v[2 * e], v[2 * e + 1]);
                v[2 * e] -= __uint_as_float(w[term][e] << 16);
                v[2 * e + 1] -= __uint_as_float(w[term][e] & 0xFFFF0000u);
            }
        uint8_t *dst = record + piece_at(t_row + r, c >> 3);
#pragma unroll
        for (int term = 0; term < 3; ++term)
            *reinterpret_cast<uint4 *>(dst + term * kTermBytes) = make_uint4(w[term][0], w[term][1], w[term][2], w[term][3]);
    }
    /* P T in tiles of 16 rows (m) and 8 columns (n), each the sum over the
     * column blocks k = n .. 2 m + 1; a warp's four tiles have 7 to 11 together */
#pragma unroll
    for (uint32_t m = 0; m < 4; ++m) {
        const uint32_t n = m == 2 ? 7 - warp : m == 1 ? warp ^ 4 : warp;
        float d[3][4] = {};
#pragma unroll
        for (uint32_t k = 0; k < 2 * m + 2; ++k)
            if (k >= n) mma_parts(d, frag_a(P, kLdP, 16 * m, 8 * k, lane), frag_b(A, kLdA, 8 * k, 8 * n, lane));
        const uint32_t col = 8 * n + 2 * (lane & 3), r = p_row + 16 * m + (lane >> 2);
        put_pair3(record, r, col, parts_sum(d, 0), parts_sum(d, 1));
        put_pair3(record, r + 8, col, parts_sum(d, 2), parts_sum(d, 3));
    }
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(128u) : "memory");
    }
}

/* ----------------------------------------------------------- second kernel */

/* k of two chunks and q of one share blocks of 192 rows: k of even chunks, q,
 * k of odd chunks. An MMA's 128 rows are then [k; q] for even chunks and [q; k]
 * for odd ones, and the lanes of an accumulator change their part likewise. */
constexpr uint32_t kBlockRows = 3 * kC;
constexpr uint32_t kBlock = kBlockRows * 128; /* bytes of 64 columns */

/* Warps: up to 16 for the epilogues (a TMEM lane and eight value rows each
 * thread), one for the MMAs, one for the records, two to load k and q. That
 * makes 20 for 32 value rows, five for each part of the SM, with 96 registers a
 * thread: at 22 they had 80, spilled the next chunk's values and so waited for
 * them (7000 cycles a chunk). */
template <int K, int VB>
struct Scan {
    static constexpr int kSubs = VB / 8;
    static constexpr int kTiles = K > 128 ? K / 128 : 1;         /* M = 128 tiles of key rows */
    /* 16 value rows leave room for warps of their own for each tile of the
     * state; the tokens are the first group's */
    static constexpr int kGroups = VB == 16 ? kTiles : 1, kOwn = kTiles / kGroups;
    static constexpr uint32_t kTokenWarps = 4 * kSubs, kEpiWarps = kTokenWarps * kGroups;
    static constexpr uint32_t kThreads = (kEpiWarps + 4) * 32, kLoadThreads = 64;
    static constexpr uint32_t kAtoms = 3 * VB > 64 ? 2 : 1;      /* blocks of 64 columns of an operand of 3 VB */
    /* With 32 value rows and keys of 256 the third term of P T has no place of
     * its own: it lies in the half of S0's second block that the third term of
     * S0 leaves free (pieces 4 to 7 of a row: its columns 0 .. 31 in the rows 0
     * .. 63, the others in the next 64 rows). */
    static constexpr bool kSplit = K == 256 && VB == 32;
    /* shared memory */
    static constexpr uint32_t kKQ = 0;
    static constexpr uint32_t kPair = kKQ + (K / 64) * kBlock;   /* terms of [T; P T] */
    static constexpr uint32_t kS = kPair + (kSplit ? 2 * kTermBytes + kC * 128 : kPairBytes); /* terms of S0, rows k */
    static constexpr uint32_t kThirdP = kS + K * 128 + 64;       /* where kSplit */
    /* terms of the scaled D and of R, rows token. The third term of 32 value
     * rows takes half of a second block: R's first, D's the other half of it. */
    static constexpr uint32_t kD = kS + kAtoms * K * 128;
    static constexpr uint32_t kR = kD + kC * 128;
    static constexpr uint32_t kDNext = kR + kC * 128 - kD;
    static constexpr uint32_t kScal = kR + kAtoms * kC * 128;    /* rows of scalars of two chunks */
    static constexpr uint32_t kBar = kScal + 2 * kScalBytes;
    static constexpr uint32_t kBad = kBar + 200;                 /* of each value row: the first token that is not finite */
    static constexpr uint32_t kBytes = kBad + VB * 4; /* the kernel has no other shared memory: its base is aligned */
    /* TMEM columns */
    static constexpr uint32_t kD1 = 0, kD3 = 4 * VB, kD3Third = kD3 + 3 * VB, kD4 = 8 * VB, kD4Tile = 4 * VB;
    static constexpr uint32_t kOThird = kSplit ? 3 * VB : kD3Third; /* the third term's product for the outputs */
    static constexpr uint32_t kColumns = 16 * VB;                /* a power of two that holds them */
};

template <int K, int VB>
__global__ void __launch_bounds__(Scan<K, VB>::kThreads, 1)
    chunk_scan_kernel(const __grid_constant__ DeltaParams p, const uint8_t *records, const uint32_t *order, uint32_t out_wide) {
    using L = Scan<K, VB>;
    constexpr int kTiles = L::kTiles;
    constexpr uint32_t kMmaWarp = L::kEpiWarps, kRecWarp = kMmaWarp + 1, kLoadWarp = kMmaWarp + 2;
    extern __shared__ __align__(1024) uint8_t sm[];
    const uint32_t base = smem_u32(sm);
    if (base & 1023u) {
        /* the swizzle would not be where the MMAs look for it */
        atomicExch(&g_chunk_status, 1);
        return;
    }
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t vblocks = p.V / VB;
    const uint32_t place = blockIdx.x / (p.HV * vblocks), rem = blockIdx.x - place * (p.HV * vblocks);
    const uint32_t h = rem / vblocks, v0 = (rem - h * vblocks) * VB, hq = h / (p.HV / p.H);
    __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(p.out) + (int64_t)h * p.out_head + v0;

    const uint32_t bar = base + L::kBar;
    const uint32_t full_kq = bar, empty_k = bar + 16, empty_q = bar + 32, full_pair = bar + 40, empty_pair = bar + 48,
                   s_ready = bar + 56, d1_full = bar + 72, r_ready = bar + 80, d3_full = bar + 88, d_ready = bar + 96,
                   d4_full = bar + 104, drain = bar + 120, full_scal = bar + 128, empty_scal = bar + 160,
                   o_full = L::kSplit ? bar + 184 : d_ready, full_third = bar + 192;
    uint32_t *slot = reinterpret_cast<uint32_t *>(sm + L::kBar + 144);
    volatile uint32_t *abort = reinterpret_cast<volatile uint32_t *>(sm + L::kBar + 152);
    volatile uint32_t *any_bad = reinterpret_cast<volatile uint32_t *>(sm + L::kBar + 176);
    uint32_t *first_bad = reinterpret_cast<uint32_t *>(sm + L::kBad);
    if (tid < (uint32_t)VB) first_bad[tid] = 0xffffffffu;
    if (tid == 0) {
        *any_bad = 0;
        for (int i = 0; i < 2; ++i) {
            mbar_init(full_scal + 8 * i, 1);
            mbar_init(empty_scal + 8 * i, L::kEpiWarps);
            mbar_init(full_kq + 8 * i, L::kLoadThreads / 32);
            mbar_init(empty_k + 8 * i, 1);
            mbar_init(s_ready + 8 * i, L::kTokenWarps);
            mbar_init(d4_full + 8 * i, 1);
        }
        mbar_init(empty_q, 1);
        mbar_init(full_pair, 1);
        mbar_init(empty_pair, 1);
        mbar_init(d1_full, 1);
        mbar_init(r_ready, L::kTokenWarps / 2);
        mbar_init(d3_full, 1);
        mbar_init(d_ready, L::kTokenWarps / 2);
        mbar_init(drain, 1);
        if (L::kSplit) {
            mbar_init(o_full, 1);
            mbar_init(full_third, 1);
        }
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)),
                     "r"(L::kColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    const uint32_t d1 = tmem + L::kD1, d3 = tmem + L::kD3, d4 = tmem + L::kD4;

    pdl_wait();
    const uint32_t n = __ldcg(order + place);
    uint32_t t0, t1;
    sequence_tokens(p, n, t0, t1);
    const int64_t pool = sequence_slot(p, n);
    const bool fresh = p.fresh != nullptr && p.fresh[n] != 0;
    float *S = p.state + (pool < 0 ? 0 : pool * p.state_slot) + ((int64_t)h * p.V + v0) * K;
    /* no chunks, no waits: only what such a sequence leaves behind */
    const uint32_t chunks = pool < 0 ? 0 : (t1 - t0 + kC - 1) / kC, rec0 = record_of(t0, n);
    if (pool < 0) {
        for (uint64_t i = tid; i < (uint64_t)(t1 - t0) * VB; i += L::kThreads)
            out[(int64_t)(t0 + i / VB) * p.out_token + i % VB] = __float2bfloat16_rn(0.0f);
    } else if (chunks == 0 && fresh) {
        for (uint32_t i = tid; i < VB * K; i += L::kThreads) S[i] = 0.0f;
    }

    if (chunks == 0) {
    } else if (warp >= kLoadWarp) {
        /* q of a chunk once the first MMAs of the chunk before have read
         * theirs, k two chunks after the same rows' last MMAs */
        const __nv_bfloat16 *q = static_cast<const __nv_bfloat16 *>(p.q) + (int64_t)hq * p.q_head;
        const __nv_bfloat16 *k = static_cast<const __nv_bfloat16 *>(p.k) + (int64_t)hq * p.k_head;
        const uint32_t th = tid - kLoadWarp * 32;
        load_rows<K, L::kLoadThreads>(base + L::kKQ, kBlock, 0, k, t0, p.k_token, min((uint32_t)kC, t1 - t0), th);
        for (uint32_t c = 0; c < chunks; ++c) {
            const uint32_t tc = t0 + c * kC;
            if (c >= 1 && !wait_bar_warp<true>(empty_q, (c - 1) & 1u, abort)) break;
            load_rows<K, L::kLoadThreads>(base + L::kKQ, kBlock, kC, q, tc, p.q_token, min((uint32_t)kC, t1 - tc), th);
            cp_async_wait_all();
            fence_async();
            warp_arrive(full_kq + 8 * (c & 1));
            if (c + 1 < chunks) {
                const uint32_t st = (c + 1) & 1, tn = tc + kC;
                if (c >= 1 && !wait_bar_warp<true>(empty_k + 8 * st, ((c - 1) >> 1) & 1u, abort)) break;
                load_rows<K, L::kLoadThreads>(base + L::kKQ, kBlock, st * 2 * kC, k, tn, p.k_token, min((uint32_t)kC, t1 - tn), th);
            }
        }
        cp_async_wait_all();
    } else if (warp == kRecWarp) {
        /* [T; P T] of a chunk once the MMAs have read that of the chunk
         * before, the next chunk's scalars once every epilogue warp has
         * read those of two chunks before it: not every one of them waits
         * for these MMAs. */
        auto expect = [&](uint32_t bytes, uint32_t full) {
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full), "r"(bytes) : "memory");
        };
        auto copy = [&](uint32_t dst, const uint8_t *src, uint32_t bytes, uint32_t full) {
            asm volatile(
                "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                "l"(src), "r"(bytes), "r"(full)
                : "memory");
        };
        auto copy_scalars = [&](const uint8_t *src, uint32_t st) {
            if (lane != 0) return;
            expect(kScalBytes, full_scal + 8 * st);
            copy(base + L::kScal + st * kScalBytes, src + kPairBytes, kScalBytes, full_scal + 8 * st);
        };
        auto copy_pair = [&](const uint8_t *src, uint32_t chunk) {
            if (lane != 0) return;
            constexpr uint32_t kThird = L::kSplit ? kC * 128 : 0;
            expect(L::kS - L::kPair, full_pair);
            if (blockIdx.x + 1 == p.drop) return;
            copy(base + L::kPair, src, L::kSplit ? 2 * kTermBytes : kPairBytes, full_pair);
            if (L::kSplit)
                copy(base + L::kPair + 2 * kTermBytes, src + 2 * kTermBytes + (chunk & 1) * kThird, kThird, full_pair);
        };
        /* the third term of P T, in the rows of the chunk's q, once the MMAs
         * have read that of the chunk before. Its pieces keep their places in the
         * swizzle; those of the columns 0 .. 31 go to the other half of the row. */
        auto copy_third = [&](const uint8_t *src, uint32_t chunk) {
            if (chunk >= 1 && !wait_bar_warp<true>(o_full, (chunk - 1) & 1u, abort)) return false;
            src += 2 * kTermBytes + (1 - (chunk & 1)) * kC * 128;
            const uint32_t dst = base + L::kThirdP - 64;
#pragma unroll 4
            for (uint32_t x = lane; x < kC * 8; x += 32) {
                const uint32_t r = x >> 3, at = x & 7, right = (at ^ r) & 4; /* where the piece lies; whether of columns 32 .. 63 */
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                                 dst + ((right ? kC : 0) + r) * 128 + ((right ? at : at ^ 4) << 4)),
                             "l"(src + x * 16)
                             : "memory");
            }
            cp_async_wait_all();
            fence_async();
            warp_arrive(full_third);
            return true;
        };
        const uint8_t *src = records + ((size_t)rec0 * p.HV + h) * kRecordBytes;
        const size_t step = (size_t)p.HV * kRecordBytes;
        uint32_t pairs = 0, scals = 1; /* copies begun */
        copy_scalars(src, 0);
        for (; pairs < chunks; src += step) {
            if (pairs >= 1 && !wait_bar_warp<true>(empty_pair, (pairs - 1) & 1u, abort)) break;
            copy_pair(src, pairs++);
            if (L::kSplit && !copy_third(src, pairs - 1)) break;
            if (pairs == chunks) break;
            const uint32_t st = scals & 1;
            if (scals >= 2 && !wait_bar_warp<true>(empty_scal + 8 * st, (scals / 2 - 1) & 1u, abort)) break;
            copy_scalars(src + step, st);
            ++scals;
        }
        /* the last copies land before the CTA ends (an abort does not stop them) */
        auto landed = [&](uint32_t x) { return mbar_try(full_scal + 8 * (x & 1), (x >> 1) & 1u); };
        const uint64_t w0 = gtimer();
        while (!((pairs == 0 || mbar_try(full_pair, (pairs - 1) & 1u)) && landed(scals - 1) &&
                 (scals == 1 || landed(scals - 2))) &&
               gtimer() - w0 < kWaitNs) {
        }
    } else if (warp == kMmaWarp) {
        /* the whole warp walks along, so that what the MMAs take stays in
         * uniform registers; one lane issues */
        const uint32_t leader = elect_one();
        const uint32_t s_desc = desc(base + L::kS, K * 128), r_desc = desc(base + L::kR, kC * 128),
                       x_desc = desc(base + L::kD, L::kDNext + 64), pair_desc = desc(base + L::kPair, 16),
                       third_desc = desc(base + L::kPair + 2 * kTermBytes, 16), third_p_desc = desc(base + L::kThirdP, 16);
        constexpr uint32_t kAll = 3 * VB, kTwo = 2 * VB;
        for (uint32_t c = 0; c < chunks; ++c) {
            const uint32_t st = c & 1, ph = c & 1;
            const uint32_t rows = base + L::kKQ + st * kC * 128;      /* [k; q] or [q; k] */
            const uint32_t k_rows = base + L::kKQ + st * 2 * kC * 128;
            if (!wait_bar_warp(full_kq + 8 * st, (c >> 1) & 1u, abort)) break;
            /* [K; Q] S0^T, 128 key rows at a time as the state's terms get ready */
            bool ok = true;
#pragma unroll
            for (int t = 0; t < kTiles && ok; ++t) {
                ok = wait_bar_warp(s_ready + 8 * t, ph, abort);
                tc_fence_after();
                if (ok && leader) {
                    const uint32_t a = desc(rows, 16);
#pragma unroll
                    for (int kk = t * (K / 16 / kTiles); kk < (t + 1) * (K / 16 / kTiles); ++kk)
                        mma(d1, a + (((kk / 4) * kBlock + (kk % 4) * 32) >> 4), s_desc + ((kk * 2048) >> 4),
                            instr_desc(128, kAll, false, true), kk != 0);
                }
            }
            if (!ok) break;
            if (leader) {
                commit(d1_full);
                commit(empty_q);
            }
            if (!wait_bar_warp(full_pair, ph, abort) || !wait_bar_warp(r_ready, ph, abort)) break;
            tc_fence_after();
            if (leader) {
                /* [T; P T] R: the first term with all of R, the second with R's first
                 * two, the third with R's first, in columns of their own. Where
                 * kSplit, T's third alone: the rows of q run into other memory and
                 * are not read, nor are those of k with P T's third, which nobody
                 * but the outputs waits for. */
#pragma unroll
                for (int kk = 0; kk < kC / 16; ++kk)
                    mma(d3, pair_desc + ((kk * 32) >> 4), r_desc + ((kk * 2048) >> 4), instr_desc(128, kAll, false, true), kk != 0);
#pragma unroll
                for (int kk = 0; kk < kC / 16; ++kk)
                    mma(d3, pair_desc + ((kTermBytes + kk * 32) >> 4), r_desc + ((kk * 2048) >> 4),
                        instr_desc(128, kTwo, false, true), true);
#pragma unroll
                for (int kk = 0; kk < kC / 16; ++kk)
                    mma(tmem + L::kD3Third, third_desc - (L::kSplit ? st * ((kC * 128) >> 4) : 0) + ((kk * 32) >> 4),
                        r_desc + ((kk * 2048) >> 4), instr_desc(128, VB, false, true), kk != 0);
                commit(d3_full);
                commit(empty_pair);
            }
            if (L::kSplit) {
                if (!wait_bar_warp(full_third, ph, abort)) break;
                tc_fence_after();
                if (leader) {
#pragma unroll
                    for (int kk = 0; kk < kC / 16; ++kk)
                        mma(tmem + L::kOThird,
                            third_p_desc + (((kk >> 1) * kC * 128 + (kk & 1) * 32) >> 4) - (1 - st) * ((kC * 128) >> 4),
                            r_desc + ((kk * 2048) >> 4), instr_desc(128, VB, false, true), kk != 0);
                    commit(o_full);
                }
            }
            if (!wait_bar_warp(d_ready, ph, abort)) break;
            tc_fence_after();
            if (leader) {
                /* K^T D (64 key rows: the upper half of M runs into other rows and is not read) */
                const uint32_t a = desc(k_rows, K >= 128 ? kBlock : kC * 128);
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
#pragma unroll
                    for (int kk = 0; kk < kC / 16; ++kk)
                        mma(d4 + L::kD4Tile * t, a + ((t * 2 * kBlock + kk * 2048) >> 4), x_desc + ((kk * 2048) >> 4),
                            instr_desc(128, kAll, true, true), kk != 0);
                    commit(d4_full + 8 * t);
                }
                commit(empty_k + 8 * st);
            }
        }
        /* every MMA issued is done before TMEM is released */
        if (leader) {
            commit(drain);
            const uint64_t w0 = gtimer();
            while (!mbar_try(drain, 0) && gtimer() - w0 < kWaitNs) {
            }
        }
    } else {
        /* epilogues: thread = TMEM lane (token of k or q, or key row) and eight
         * of the value rows */
        const uint32_t ln = 32 * (warp & 3) + lane, sub = (warp >> 2) % L::kSubs, group = warp / L::kTokenWarps;
        const uint32_t at = ((32 * (warp & 3)) << 16) + 8 * sub;
        const uint32_t i = ln & (kC - 1);
        const __nv_bfloat16 *v = static_cast<const __nv_bfloat16 *>(p.v) + (int64_t)h * p.v_head + v0 + 8 * sub;
        const bool has_s = K >= 128 || ln < (uint32_t)K;
        const uint32_t tile0 = group * L::kOwn; /* this warp's tiles of the state */
        float s[L::kOwn][8];
#pragma unroll
        for (int t = 0; t < L::kOwn; ++t)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                s[t][e] = (has_s && !fresh) ? S[(int64_t)(8 * sub + e) * K + 128 * (tile0 + t) + ln] : 0.0f;
        /* in a chunk, whether this lane is a token of q (uniform in a warp) */
        auto is_q = [&](uint32_t c) { return (ln >= (uint32_t)kC) != ((c & 1) != 0); };
        /* the lane's value rows of a chunk, requested one chunk ahead */
        uint4 next = make_uint4(0, 0, 0, 0);
        auto fetch = [&](uint32_t c) {
            const uint32_t t = t0 + c * kC + i;
            next = make_uint4(0, 0, 0, 0);
            if (!is_q(c) && t < t1) next = *reinterpret_cast<const uint4 *>(v + (int64_t)t * p.v_token);
        };
        fetch(0);
#pragma unroll
        for (int t = 0; t < L::kOwn; ++t) {
            if (has_s) put_terms<VB>(sm + L::kS, K * 128, 128 * (tile0 + t) + ln, sub, s[t]);
            fence_async();
            warp_arrive(s_ready + 8 * (tile0 + t));
        }
        bool ok = true;
        for (uint32_t c = 0; c < chunks; ++c) {
            const uint32_t ph = c & 1, tc = t0 + c * kC, rows = min((uint32_t)kC, t1 - tc);
            const bool q = is_q(c);
            const float *sc = reinterpret_cast<const float *>(sm + L::kScal + ph * kScalBytes);
            if (!(ok = wait_bar_warp(full_scal + 8 * ph, (c >> 1) & 1u, abort))) break;
            const float decay = sc[kScalDecay * kC], f2 = sc[kScalEnd * kC + i];
            /* the decayed state, and beta v, do not wait for the MMAs */
#pragma unroll
            for (int t = 0; t < L::kOwn; ++t)
#pragma unroll
                for (int e = 0; e < 8; ++e) s[t][e] *= decay;
            float x[8];
            if (group == 0) {
                float bv[8], f0;
                uint32_t poison = 0; /* value rows of this token that are not finite */
                if (q) {
                    f0 = sc[kScalQ * kC + i];
                } else {
                    const float beta = sc[kScalBeta * kC + i];
                    const uint32_t u[4] = {next.x, next.y, next.z, next.w};
                    f0 = -beta * sc[kScalC * kC + i];
#pragma unroll
                    for (int e = 0; e < 8; ++e) bv[e] = beta * __uint_as_float((e & 1) ? (u[e >> 1] & 0xFFFF0000u) : (u[e >> 1] << 16));
                }
                warp_arrive(empty_scal + 8 * ph);
                if (c + 1 < chunks) fetch(c + 1);
                float o[8];
                if (!(ok = wait_bar_warp(d1_full, ph, abort))) break;
                tc_fence_after();
                tc_sum3<VB>(d1 + at, x);
                if (q) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[e] = f0 * x[e];
                } else {
                    /* rows without a token have zeros for all of it */
                    scale_add(f0, x, bv);
                    put_terms<VB>(sm + L::kR, kC * 128, i, sub, bv);
                    if (!all_finite(bv)) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (!(bv[e] * 0.0f == 0.0f)) {
                                bv[e] = 0.0f;
                                poison |= 1u << e;
                                atomicMin(first_bad + 8 * sub + e, c * kC + i);
                            }
                        *any_bad = 1;
                        put_terms<VB>(sm + L::kR, kC * 128, i, sub, bv);
                    }
                    fence_async();
                    tc_fence_before();
                    warp_arrive(r_ready);
                }
                /* the outputs' rows let those of D go first, which the state waits
                 * for (4096 tokens 168.7 us, both at once 170.4) */
                if (!(ok = wait_bar_warp(q ? o_full : d3_full, ph, abort))) break;
                tc_fence_after();
                tc_sum3<VB>(d3 + at, x);
                uint32_t third[8];
                __syncwarp();
                tc_ld8(tmem + (q ? L::kOThird : L::kD3Third) + at, third);
                tc_wait();
                if (q) {
                    if (i < rows) {
                        __nv_bfloat16 *dst = out + (int64_t)(tc + i) * p.out_token + 8 * sub;
#pragma unroll
                        for (int e = 0; e < 8; ++e) o[e] += x[e] + __uint_as_float(third[e]);
                        if (*any_bad) {
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                if (c * kC + i >= first_bad[8 * sub + e]) o[e] = __int_as_float(0x7fc00000);
                        }
                        if (out_wide) {
                            *reinterpret_cast<uint4 *>(dst) = make_uint4(bf16_pair(o[0], o[1]), bf16_pair(o[2], o[3]),
                                                                         bf16_pair(o[4], o[5]), bf16_pair(o[6], o[7]));
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e) dst[e] = __float2bfloat16_rn(o[e]);
                        }
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = f2 * (x[e] + __uint_as_float(third[e]));
                    if (poison) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if ((poison >> e) & 1u) x[e] = __int_as_float(0x7fc00000);
                    }
                    put_terms<VB, 4>(sm + L::kD, L::kDNext, i, sub, x);
                    fence_async();
                    tc_fence_before();
                    warp_arrive(d_ready);
                }
            } else {
                warp_arrive(empty_scal + 8 * ph);
            }
#pragma unroll
            for (int t = 0; t < L::kOwn; ++t) {
                if (!(ok = wait_bar_warp(d4_full + 8 * (tile0 + t), ph, abort))) break;
                tc_fence_after();
                tc_sum3<VB>(d4 + L::kD4Tile * (tile0 + t) + at, x);
                add_to(x, s[t]);
                if (c + 1 < chunks) {
                    if (has_s) put_terms<VB>(sm + L::kS, K * 128, 128 * (tile0 + t) + ln, sub, s[t]);
                    fence_async();
                    tc_fence_before();
                    warp_arrive(s_ready + 8 * (tile0 + t));
                }
            }
            if (!ok) break;
        }
        if (has_s) {
            /* a sequence that was given up leaves no state that could pass for one */
            const float bad = __int_as_float(0x7fc00000);
#pragma unroll
            for (int t = 0; t < L::kOwn; ++t)
#pragma unroll
                for (int e = 0; e < 8; ++e) S[(int64_t)(8 * sub + e) * K + 128 * (tile0 + t) + ln] = ok ? s[t][e] : bad;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kColumns) : "memory");
    }
}

/* bytes of the order of N sequences, before the records */
size_t order_bytes(uint32_t sequences) { return ((size_t)sequences * 4 + 255) & ~(size_t)255; }
uint32_t record_count(uint32_t tokens, uint32_t sequences) { return tokens / kC + sequences + 2; }

template <int K, int VB>
cudaError_t launch_scan(const DeltaParams &p, const uint8_t *records, const uint32_t *order, cudaStream_t stream) {
    using L = Scan<K, VB>;
    cudaError_t e = cudaFuncSetAttribute(chunk_scan_kernel<K, VB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kBytes);
    if (e != cudaSuccess) return e;
    const uint32_t wide = (reinterpret_cast<uintptr_t>(p.out) & 15) == 0 && p.out_token % 8 == 0 && p.out_head % 8 == 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.N * p.HV * (p.V / VB));
    cfg.blockDim = dim3(L::kThreads);
    cfg.dynamicSmemBytes = L::kBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, chunk_scan_kernel<K, VB>, p, records, order, wide);
}

template <int K>
cudaError_t launch_chunk_k(const DeltaParams &p, uint8_t *workspace, int sms, cudaStream_t stream) {
    uint32_t *order = reinterpret_cast<uint32_t *>(workspace);
    uint8_t *records = workspace + order_bytes(p.N);
    cudaError_t e = cudaFuncSetAttribute(chunk_prep_kernel<K>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)PrepSmem<K>::kBytes);
    if (e != cudaSuccess) return e;
    e = launch(chunk_prep_kernel<K>, dim3(record_count(p.tokens, p.N), p.HV), kPrepThreads, PrepSmem<K>::kBytes, stream, p, records,
               order);
    if (e != cudaSuccess) return e;
    const uint32_t ctas16 = p.N * p.HV * (p.V / 16);
    if (ctas16 > (uint32_t)sms) return launch_scan<K, 32>(p, records, order, stream);
    return launch_scan<K, 16>(p, records, order, stream);
}

}  // namespace

size_t delta_chunk_workspace(uint32_t tokens, uint32_t sequences, uint32_t v_heads) {
    return order_bytes(sequences) + (size_t)record_count(tokens, sequences) * v_heads * kRecordBytes;
}

cudaError_t launch_delta_chunk(const DeltaParams &p, void *workspace, int sms, cudaStream_t stream) {
    uint8_t *w = static_cast<uint8_t *>(workspace);
    switch (p.K) {
        case 64: return launch_chunk_k<64>(p, w, sms, stream);
        case 128: return launch_chunk_k<128>(p, w, sms, stream);
        default: return launch_chunk_k<256>(p, w, sms, stream);
    }
}

cudaError_t delta_chunk_status(int *status) {
    cudaError_t e = cudaMemcpyFromSymbol(status, g_chunk_status, sizeof(int));
    const int zero = 0;
    if (e == cudaSuccess && *status != 0) e = cudaMemcpyToSymbol(g_chunk_status, &zero, sizeof(int));
    return e;
}

}  // namespace ops
}  // namespace gdn
