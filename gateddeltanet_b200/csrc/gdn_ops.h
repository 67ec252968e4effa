/* Internal interface between the C entries of the serving operators
 * (gdn_ops_host.cu) and their kernels: the gated delta rule over pooled
 * states (gdn_delta.cu, gdn_delta_chunk.cu), the constraints on logits
 * (gdn_logits.cu), norms (gdn_norm.cu), the short convolution (gdn_conv.cu) and
 * projections (gdn_linear.cu, gdn_linear_few.cu). Device pointers throughout;
 * strides count elements. Not installed; callers use include/gdn_b200.h. */
#ifndef GDN_OPS_H
#define GDN_OPS_H

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace gdn {
namespace ops {

/* Packed tokens of N sequences: sequence n has the tokens starts[n] ..
 * starts[n + 1] - 1 (starts null: token n alone). */
struct DeltaParams {
    const void *q, *k, *v;
    const float *g, *beta;
    float *state;
    void *out;
    const int32_t *starts, *slots;
    const uint8_t *fresh;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head;
    int64_t g_token, g_head, beta_token, beta_head, out_token, out_head, state_slot;
    uint32_t N, tokens, H, HV, K, V, state_slots;
    int normalize;
    float scale;
    uint32_t drop; /* for tests, 0: none. 1 + the row block (pipeline) or CTA (chunks) whose copy is not made */
};

/* Tokens [t0, t1) of sequence n, clamped to the packed tensors so that no
 * content of starts leads out of them. */
__host__ __device__ __forceinline__ void sequence_tokens(const DeltaParams &p, uint32_t n, uint32_t &t0, uint32_t &t1) {
    if (p.starts == nullptr) {
        t0 = n;
        t1 = n + 1;
        return;
    }
    const int32_t a = p.starts[n], b = p.starts[n + 1];
    t0 = a < 0 ? 0u : ((uint32_t)a < p.tokens ? (uint32_t)a : p.tokens);
    t1 = b < 0 ? 0u : ((uint32_t)b < p.tokens ? (uint32_t)b : p.tokens);
    if (t1 < t0) t1 = t0;
}

/* Tokens [first, end) from the first sequence's begin to the last one's end,
 * and the walk over the others, which belong to no sequence. Never end < first,
 * so that the walk moves forward whatever starts holds. */
struct Covered {
    uint32_t first, end;
    __host__ __device__ __forceinline__ uint32_t first_outside() const { return first == 0 ? end : 0; }
    __host__ __device__ __forceinline__ uint32_t next_outside(uint32_t t) const { return t + 1 == first ? end : t + 1; }
};
__host__ __device__ __forceinline__ Covered covered_tokens(const DeltaParams &p) {
    uint32_t first, t0, t1, last;
    sequence_tokens(p, 0, first, t0);
    sequence_tokens(p, p.N - 1, t1, last);
    return {first, last < first ? first : last};
}

/* Pool slot of sequence n; negative if it has none (its tokens then give
 * zeros and no state changes). */
__device__ __forceinline__ int64_t sequence_slot(const DeltaParams &p, uint32_t n) {
    const int64_t s = p.slots == nullptr ? (int64_t)n : (int64_t)p.slots[n];
    return s < (int64_t)p.state_slots ? s : -1;
}

struct LogitsParams {
    const void *logits;
    void *out;
    int32_t *picks;
    const int32_t *tokens, *lens, *prompt_lens;
    const float *repetition, *presence, *frequency;
    const int32_t *bias_ids;
    const float *bias;
    const uint32_t *mask;
    int64_t logits_row, out_row, tokens_row, bias_ids_row, bias_row, mask_row;
    uint32_t rows, vocab, history, biases;
    uint32_t slice_vecs;  /* 16-byte vectors of a row that one CTA takes */
};

constexpr uint32_t kMaxHistory = (1u << 20) - 1;
constexpr uint32_t kMaxBiases = 2047;  /* searched once for each biased token */
constexpr uint32_t kMaxVocab = 1u << 18;

/* Codes of element types, as in include/gdn_b200.h. */
enum Type : int { kF32 = 0, kBF16 = 1, kE4M3 = 2 };

/* Rows of heads x dim; what is absent is null. */
struct NormParams {
    const void *x, *gate, *weight;
    void *residual, *out;
    float *scales;
    int64_t x_token, x_head, gate_token, gate_head, residual_token, residual_head, out_token, out_head;
    uint32_t tokens, heads, dim;
    int type, weight_type, residual_type, out_type;
    float eps;
};
constexpr uint32_t kMaxNormThreads = 1024;
/* Threads of a row of dim values, `each` to a thread: a power of two up to 32, or a multiple of 32. */
inline uint32_t norm_group(uint32_t dim, uint32_t each) {
    const uint32_t need = dim / each + (dim % each != 0);
    if (need > 32) return (need + 31) / 32 * 32;
    uint32_t group = 1;
    while (group < need) group *= 2;
    return group;
}
/* Threads that have to be in one CTA: a row's, or those of all heads of a token with one scale. */
inline uint64_t norm_threads(const NormParams &p, uint32_t each) {
    return (uint64_t)norm_group(p.dim, each) * (p.out_type == 2 ? p.heads : 1);
}

/* Packed tokens of N sequences, as in DeltaParams. */
struct ConvParams {
    const void *x, *weight, *bias;
    void *tails, *out;
    const int32_t *starts, *slots;
    const uint8_t *fresh;
    int64_t x_token, out_token, tails_slot, tails_row;
    uint32_t N, tokens, channels, width, tail_slots;
    int type, weight_type, tail_type, silu;
};

/* What the walk over a tile [t0, t1), come to token t in it, does with the sequence that has the entries `bound` and
 * `end` of starts (end > t, both clamped): its tokens [t, stop) here, none if they are equal. The tile in which a sequence
 * begins takes its first `back` tokens (which meet the slot's rows) also where they lie behind the tile's end, and the tiles
 * after it leave them out. Where starts do not decrease a bound in the tile is t itself; where they do, it may be before
 * or behind t, and the sequence is taken to begin at t. So t of a sequence that does not begin here is never below
 * `back`: the rows before it that its first outputs read are in the tensor whatever starts holds. */
struct ConvPart {
    uint32_t t, stop;
    bool begins;
};
__host__ __device__ __forceinline__ ConvPart conv_part(uint32_t bound, uint32_t end, uint32_t t, uint32_t t0, uint32_t t1, uint32_t back) {
    if (bound >= t0) {
        const uint32_t least = t1 > t + back ? t1 : t + back;
        return {t, end < least ? end : least, true};
    }
    const uint32_t first = bound + back < end ? bound + back : end, from = t > first ? t : first, stop = end < t1 ? end : t1;
    return {from, stop > from ? stop : from, false};
}

enum Activation : int { kNoActivation = 0, kSilu = 1, kGelu = 2, kSwiglu = 3 };

/* y = act(sx sw x W^T + bias) + residual; W has 2 x outputs rows for kSwiglu. */
struct LinearParams {
    const void *x, *weight, *bias, *residual;
    const float *x_scales, *weight_scales;
    void *out;
    int64_t x_row, weight_row, residual_row, out_row;
    uint32_t tokens, inputs, outputs;
    int type, bias_type, residual_type, out_type, activation;
    uint32_t drop; /* for tests, 0: none. 1 + the k-block whose copy the first CTA does not make */
    uint32_t tiles; /* for tests, 0: those of the rule. CTAs to a tile, columns << 4 and CTAs that divide k << 16 */
};
constexpr uint32_t kFewTokens = 16; /* that gdn_linear_few.cu can take */

/* kernel<<<grid, block, smem, stream>>>(args...) and this launch's own result:
 * cudaGetLastError would also give that of a call before it. */
template <typename... Params, typename... Args>
cudaError_t launch(void (*kernel)(Params...), dim3 grid, uint32_t block, size_t smem, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

/* the same for a kernel that begins with wait_for_previous(), so that its launch and set-up overlap the
 * end of the kernel before it */
template <typename... Params, typename... Args>
cudaError_t launch_overlapped(void (*kernel)(Params...), dim3 grid, uint32_t block, size_t smem, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

cudaError_t launch_delta_step(const DeltaParams &p, bool bf16, int sms, cudaStream_t stream);
/* The chunked form (gdn_delta_chunk.cu): BF16, 16-byte aligned rows. */
size_t delta_chunk_workspace(uint32_t tokens, uint32_t sequences, uint32_t v_heads);
cudaError_t launch_delta_chunk(const DeltaParams &p, void *workspace, int sms, cudaStream_t stream);
/* *status != 0: a wait of such a kernel on the current device ran out since
 * the last call. For kernels that have ended. */
cudaError_t delta_step_status(int *status);
cudaError_t delta_chunk_status(int *status);
cudaError_t launch_logits(LogitsParams p, bool bf16, int sms, cudaStream_t stream);
cudaError_t launch_norm(const NormParams &p, int sms, cudaStream_t stream);
cudaError_t launch_conv(const ConvParams &p, int sms, cudaStream_t stream);
cudaError_t launch_linear(const LinearParams &p, int sms, cudaStream_t stream);
bool takes_few(const LinearParams &p); /* whether launch_linear_few is the faster one */
cudaError_t launch_linear_few(const LinearParams &p, int sms, cudaStream_t stream);
cudaError_t linear_status(int *status);

}  // namespace ops
}  // namespace gdn

#endif
