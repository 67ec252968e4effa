/* Internal interface between the C entries of the serving operators
 * (gdn_ops_host.cu) and their kernels: the gated delta rule over pooled
 * states (gdn_delta.cu) and the constraints on logits (gdn_logits.cu). Device
 * pointers throughout; strides count elements. Not installed; callers use
 * include/gdn_b200.h. */
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

cudaError_t launch_delta_step(const DeltaParams &p, bool bf16, int sms, cudaStream_t stream);
/* The chunked form (gdn_delta_chunk.cu): BF16, 16-byte aligned rows. */
size_t delta_chunk_workspace(uint32_t tokens, uint32_t sequences, uint32_t v_heads);
cudaError_t launch_delta_chunk(const DeltaParams &p, void *workspace, int sms, cudaStream_t stream);
/* *status != 0: a wait of such a kernel on the current device ran out since
 * the last call. For kernels that have ended. */
cudaError_t delta_step_status(int *status);
cudaError_t delta_chunk_status(int *status);
cudaError_t launch_logits(LogitsParams p, bool bf16, int sms, cudaStream_t stream);

}  // namespace ops
}  // namespace gdn

#endif
