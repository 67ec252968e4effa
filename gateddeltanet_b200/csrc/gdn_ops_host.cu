/* gdn_ops_host.cu -- C entries of the serving operators (include/gdn_b200.h):
 * the checks of their arguments and the launches. Device pointers on the
 * caller's stream; nothing is allocated or synchronised. */
#include "gdn_b200.h"
#include "gdn_ops.h"

#include <atomic>
#include <stdarg.h>
#include <stdio.h>

namespace gdn {
int host_fail(const char *msg); /* gdn_host.cu: records the message, returns -1 */
}

namespace {

int failf(const char *fmt, ...) {
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return gdn::host_fail(buf);
}

/* A CUDA call that failed is reported here and leaves no error behind that a later check would take for its own. */
int cuda_failf(const char *who, const char *what, cudaError_t e) {
    cudaGetLastError();
    return failf("%s: %s: %s", who, what, cudaGetErrorString(e));
}

bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

/* Whether two tables of `rows` rows of `width` bytes share memory, other than
 * row by row in the same place. Strides are not negative. */
bool partly_shared(const void *x, int64_t x_row, const void *y, int64_t y_row, int64_t rows, int64_t width) {
    const int64_t d = (int64_t)(reinterpret_cast<uintptr_t>(y) - reinterpret_cast<uintptr_t>(x));
    if (rows == 1) x_row = y_row = width;
    if (d >= (rows - 1) * x_row + width || -d >= (rows - 1) * y_row + width) return false;
    if (x_row != y_row || x_row < width) return true;
    const int64_t shift = (d % x_row + x_row) % x_row; /* of y's rows against x's */
    return d != 0 && (shift < width || shift + width > x_row);
}

/* The call's device for the thread, and the previous one afterwards. */
struct DeviceScope {
    int prev = -1;
    cudaError_t error;
    explicit DeviceScope(int device) {
        error = cudaGetDevice(&prev);
        if (error != cudaSuccess || prev == device)
            prev = -1;
        else
            error = cudaSetDevice(device);
    }
    ~DeviceScope() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

cudaError_t sm_count(int device, int &sms) {
    static std::atomic<int> counts[64]; /* 0: not asked yet; every writer writes the same value */
    if (device < 0 || device >= 64) return cudaErrorInvalidDevice;
    sms = counts[device].load(std::memory_order_relaxed);
    if (sms != 0) return cudaSuccess;
    const cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess) counts[device].store(sms, std::memory_order_relaxed);
    return e;
}

/* launch(sms) on `device` */
template <typename F>
int on_device(const char *who, int device, F launch) {
    DeviceScope scope(device);
    int sms = 0;
    cudaError_t e = scope.error;
    if (e == cudaSuccess) e = sm_count(device, sms);
    if (e != cudaSuccess) return cuda_failf(who, "cannot use the device", e);
    e = launch(sms);
    return e == cudaSuccess ? 0 : cuda_failf(who, "launch failed", e);
}

std::atomic<uint32_t> g_drop{0}; /* gdn_b200_test_drop_copy */

/* Checks what both forms of the rule ask of their arguments; > 0: nothing to do. */
int delta_params(const char *who, const GdnB200DeltaArgs *a, gdn::ops::DeltaParams &p) {
    if (a == nullptr) return failf("%s: no arguments", who);
    if (a->dtype != 0 && a->dtype != 1) return failf("%s: dtype %d is neither FP32 (0) nor BF16 (1)", who, a->dtype);
    if (a->key_dim != 64 && a->key_dim != 128 && a->key_dim != 256)
        return failf("%s: key_dim %u is not 64, 128 or 256", who, a->key_dim);
    if (a->value_dim == 0 || a->value_dim > 256 || a->value_dim % 32 != 0)
        return failf("%s: value_dim %u is not a multiple of 32 up to 256", who, a->value_dim);
    if (a->heads == 0 || a->v_heads == 0 || a->v_heads % a->heads != 0 || a->v_heads > 65535)
        return failf("%s: %u value heads do not share %u query/key heads evenly", who, a->v_heads, a->heads);
    if (a->tokens > 0x7fffffffu || a->sequences > 0x3fffffu)
        return failf("%s: %u tokens in %u sequences are too many", who, a->tokens, a->sequences);
    if (((uint64_t)a->sequences + 1) * a->v_heads * (a->value_dim / 16) > 0x7fffffffu)
        return failf("%s: %u sequences of %u heads are too many", who, a->sequences, a->v_heads);
    if (a->starts == nullptr && a->tokens != a->sequences)
        return failf("%s: without starts every sequence has one token (%u tokens, %u sequences)", who, a->tokens,
                     a->sequences);
    if (a->sequences == 0) {
        if (a->tokens != 0) return failf("%s: %u tokens but no sequence", who, a->tokens);
        return 1;
    }
    if (a->slots == nullptr && a->state_slots < a->sequences)
        return failf("%s: %u state slots for %u sequences", who, a->state_slots, a->sequences);
    if (a->state == nullptr || !aligned(a->state, 16))
        return failf("%s: state is missing or not on a 16-byte boundary", who);
    const int64_t slot = (int64_t)a->v_heads * a->value_dim * a->key_dim;
    if (a->state_slot % 4 != 0 || (a->state_slot < slot && a->state_slots > 1))
        return failf("%s: state slots overlap or leave the 16-byte boundary (stride %lld)", who,
                     (long long)a->state_slot);
    if (a->tokens != 0 && (a->q == nullptr || a->k == nullptr || a->v == nullptr || a->g == nullptr ||
                           a->beta == nullptr || a->out == nullptr))
        return failf("%s: q, k, v, g, beta or out is missing", who);
    p = gdn::ops::DeltaParams{a->q, a->k, a->v, a->g, a->beta, a->state, a->out, a->starts, a->slots, a->fresh,
                              a->q_token, a->q_head, a->k_token, a->k_head, a->v_token, a->v_head,
                              a->g_token, a->g_head, a->beta_token, a->beta_head, a->out_token, a->out_head,
                              a->state_slot, a->sequences, a->tokens, a->heads, a->v_heads, a->key_dim,
                              a->value_dim, a->state_slots, a->normalize != 0, a->scale, g_drop.exchange(0)};
    return 0;
}

}  // namespace

extern "C" {

int gdn_b200_delta_step(const GdnB200DeltaArgs *args) {
    gdn::ops::DeltaParams p;
    const int rc = delta_params("gdn_b200_delta_step", args, p);
    if (rc != 0) return rc > 0 ? 0 : -1;
    return on_device("gdn_b200_delta_step", args->device, [&](int sms) {
        return gdn::ops::launch_delta_step(p, args->dtype == 1, sms, static_cast<cudaStream_t>(args->stream));
    });
}

size_t gdn_b200_delta_chunk_workspace(uint32_t tokens, uint32_t sequences, uint32_t v_heads) {
    return gdn::ops::delta_chunk_workspace(tokens, sequences, v_heads);
}

int gdn_b200_delta_status(int device) {
    DeviceScope scope(device);
    int step = 0, chunk = 0;
    cudaError_t e = scope.error;
    if (e == cudaSuccess) e = cudaDeviceSynchronize(); /* the copies below wait for no stream but their own */
    if (e == cudaSuccess) e = gdn::ops::delta_step_status(&step);
    if (e == cudaSuccess) e = gdn::ops::delta_chunk_status(&chunk);
    if (e != cudaSuccess) return cuda_failf("gdn_b200_delta_status", "cannot read the device", e);
    return step == 0 && chunk == 0 ? 0
                                   : failf("gdn_b200_delta_%s: a wait on the device ran out; the call's states are not valid",
                                           chunk != 0 ? "chunk" : "step");
}

int gdn_b200_test_drop_copy(uint32_t index) {
    g_drop = index + 1;
    return 0;
}

int gdn_b200_delta_chunk(const GdnB200DeltaArgs *args) {
    gdn::ops::DeltaParams p;
    const int rc = delta_params("gdn_b200_delta_chunk", args, p);
    if (rc != 0) return rc > 0 ? 0 : -1;
    if (args->dtype != 1)
        return failf("gdn_b200_delta_chunk: q, k and v must be BF16 (gdn_b200_delta_step takes FP32 of any length)");
    if (!aligned(args->q, 16) || !aligned(args->k, 16) || !aligned(args->v, 16) || args->q_token % 8 != 0 ||
        args->q_head % 8 != 0 || args->k_token % 8 != 0 || args->k_head % 8 != 0 || args->v_token % 8 != 0 ||
        args->v_head % 8 != 0)
        return failf("gdn_b200_delta_chunk: rows of q, k and v must start on 16-byte boundaries");
    const size_t need = gdn::ops::delta_chunk_workspace(args->tokens, args->sequences, args->v_heads);
    if (args->workspace == nullptr || !aligned(args->workspace, 256) || args->workspace_bytes < need)
        return failf("gdn_b200_delta_chunk: a workspace of %zu bytes on a 256-byte boundary is needed", need);
    return on_device("gdn_b200_delta_chunk", args->device, [&](int sms) {
        return gdn::ops::launch_delta_chunk(p, args->workspace, sms, static_cast<cudaStream_t>(args->stream));
    });
}

int gdn_b200_constrain_logits(const GdnB200LogitsArgs *args) {
    const char *who = "gdn_b200_constrain_logits";
    if (args == nullptr) return failf("%s: no arguments", who);
    const GdnB200LogitsArgs &a = *args;
    if (a.dtype != 0 && a.dtype != 1) return failf("%s: dtype %d is neither FP32 (0) nor BF16 (1)", who, a.dtype);
    if (a.rows == 0) return 0;
    if (a.rows > 0xffffffu) return failf("%s: %u rows are too many", who, a.rows);
    if (a.vocab == 0 || a.vocab > gdn::ops::kMaxVocab)
        return failf("%s: vocab %u is not in 1 .. %u", who, a.vocab, gdn::ops::kMaxVocab);
    if (a.history > gdn::ops::kMaxHistory)
        return failf("%s: a history of %u tokens is longer than %u", who, a.history, gdn::ops::kMaxHistory);
    if (a.biases > gdn::ops::kMaxBiases)
        return failf("%s: %u biases a row are more than %u", who, a.biases, gdn::ops::kMaxBiases);
    if (a.logits == nullptr || a.out == nullptr || a.picks == nullptr)
        return failf("%s: logits, out or picks is missing", who);
    if (a.tokens == nullptr && a.history != 0) return failf("%s: tokens is missing", who);
    if ((a.bias_ids == nullptr) != (a.bias == nullptr)) return failf("%s: bias_ids and bias go together", who);
    const uintptr_t elem = a.dtype == 1 ? 2 : 4;
    if (!aligned(a.logits, elem) || !aligned(a.out, elem)) return failf("%s: logits or out is misaligned", who);
    if (a.rows > 1 && a.out_row < (int64_t)a.vocab) return failf("%s: rows of out overlap", who);
    if (a.logits_row < 0) return failf("%s: negative row stride", who);
    if (partly_shared(a.logits, a.logits_row * (int64_t)elem, a.out, a.out_row * (int64_t)elem, a.rows, a.vocab * (int64_t)elem))
        return failf("%s: out overlaps logits without being logits", who);
    gdn::ops::LogitsParams p{a.logits, a.out, a.picks, a.history ? a.tokens : nullptr, a.lens, a.prompt_lens,
                             a.repetition, a.presence, a.frequency, a.biases ? a.bias_ids : nullptr, a.bias, a.mask,
                             a.logits_row, a.out_row, a.tokens_row, a.bias_ids_row, a.bias_row, a.mask_row,
                             a.rows, a.vocab, a.history, a.biases, 0};
    return on_device(who, a.device, [&](int sms) {
        return gdn::ops::launch_logits(p, a.dtype == 1, sms, static_cast<cudaStream_t>(a.stream));
    });
}

}  // extern "C"
