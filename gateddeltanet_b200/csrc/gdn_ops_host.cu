/* gdn_ops_host.cu -- C entries of the serving operators (include/gdn_b200.h):
 * the checks of their arguments and the launches. Device pointers on the
 * caller's stream; nothing is allocated or synchronised. */
#include "gdn_b200.h"
#include "gdn_ops.h"

#include <atomic>
#include <cmath>
#include <initializer_list>
#include <numeric>
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

/* Whether rows [tokens][heads] of dim values share memory (strides not negative). */
bool rows_overlap(int64_t token, int64_t head, uint32_t tokens, uint32_t heads, uint32_t dim) {
    int64_t inner = head, outer = token;
    uint32_t n_inner = heads, n_outer = tokens;
    if (heads == 1 || (tokens > 1 && token < head)) inner = token, outer = head, n_inner = tokens, n_outer = heads;
    int64_t reach = dim;
    if (n_inner > 1) {
        if (inner < reach) return true;
        reach += (n_inner - 1) * inner;
    }
    return n_outer > 1 && outer < reach;
}

std::atomic<uint32_t> g_drop{0};  /* gdn_b200_test_drop_copy */
std::atomic<uint32_t> g_tiles{0}; /* gdn_b200_test_linear_tiles */

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

bool float_type(int t) { return t == 0 || t == 1; }
int64_t size_of(int type) { return type == 0 ? 4 : type == 1 ? 2 : 1; }

/* The memory of a tensor [tokens][heads][dim], by token: from `at` on, `width`
 * bytes (with the gaps between its heads) every `row` bytes; and by runs of `run`
 * bytes, whose distances are multiples of `period` (0: there is one run). */
struct Extent {
    const void *at;
    int64_t row, width, rows, run, period;
    Extent(const void *p, int64_t token, int64_t head, uint32_t tokens, uint32_t heads, uint32_t dim, int64_t size)
        : at(p), row(token * size), width((((int64_t)heads - 1) * head + dim) * size), rows(tokens), run(dim * size), period(0) {
        if (heads > 1 && head == (int64_t)dim)
            run = width; /* heads without gaps */
        else if (heads > 1)
            period = head * size;
        if (tokens > 1) period = std::gcd(period, row);
        if (rows > 1 && row < width) { /* heads further apart than tokens: taken as one block */
            width += (rows - 1) * row;
            rows = 1;
        }
    }
    bool same(const Extent &e) const { return at == e.at && (rows == 1 || row == e.row) && width == e.width && rows == e.rows; }
    /* Whether the runs of either lie in the gaps of the other: every run of e begins `shift` bytes, and a multiple of the
     * common period, from one of these. */
    bool interleaved(const Extent &e, int64_t d) const {
        const int64_t common = std::gcd(period, e.period);
        if (common == 0) return false;
        const int64_t shift = (d % common + common) % common;
        return shift >= run && shift + e.run <= common;
    }
    bool meets(const Extent &e) const {
        if (at == nullptr || e.at == nullptr || width <= 0 || e.width <= 0) return false;
        const int64_t d = (int64_t)(reinterpret_cast<uintptr_t>(e.at) - reinterpret_cast<uintptr_t>(at));
        if (interleaved(e, d)) return false;
        if (width == e.width && rows == e.rows) return same(e) || partly_shared(at, row, e.at, e.row, rows, width);
        if (d >= (rows - 1) * row + width || -d >= (e.rows - 1) * e.row + e.width) return false;
        if (rows != e.rows || rows == 1 || row != e.row || row < width || row < e.width) return true;
        const int64_t shift = (d % row + row) % row; /* of e's rows against these */
        return shift < width || shift + e.width > row;
    }
};

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

int gdn_b200_test_linear_tiles(uint32_t ctas, uint32_t columns, uint32_t split) {
    if (ctas > 15 || columns > 4095 || split > 65535) return failf("gdn_b200_test_linear_tiles: no such tiles");
    g_tiles = ctas | columns << 4 | split << 16;
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

int gdn_b200_rms_norm(const GdnB200NormArgs *args) {
    const char *who = "gdn_b200_rms_norm";
    if (args == nullptr) return failf("%s: no arguments", who);
    const GdnB200NormArgs &a = *args;
    if (!float_type(a.dtype)) return failf("%s: dtype %d is neither FP32 (0) nor BF16 (1)", who, a.dtype);
    if (a.weight != nullptr && !float_type(a.weight_dtype)) return failf("%s: weight_dtype %d is neither FP32 (0) nor BF16 (1)", who, a.weight_dtype);
    if (a.residual != nullptr && !float_type(a.residual_dtype))
        return failf("%s: residual_dtype %d is neither FP32 (0) nor BF16 (1)", who, a.residual_dtype);
    if (!float_type(a.out_dtype) && a.out_dtype != 2) return failf("%s: out_dtype %d is not FP32 (0), BF16 (1) or E4M3 (2)", who, a.out_dtype);
    if (a.tokens == 0 || (a.heads == 0 && a.out_dtype != 2)) return 0;
    if (a.dim == 0 || a.heads == 0) return failf("%s: rows of no values", who); /* without heads a token's scale says nothing */
    if ((uint64_t)a.tokens * a.heads > 0x7fffffffu) return failf("%s: %u tokens of %u heads are too many", who, a.tokens, a.heads);
    if (!(a.eps >= 0.0f) || std::isinf(a.eps)) return failf("%s: eps is negative or not finite", who);
    if (a.x == nullptr || a.out == nullptr) return failf("%s: x or out is missing", who);
    if (a.out_dtype == 2 && a.scales == nullptr) return failf("%s: scales is missing", who);
    for (int64_t stride : {a.x_token, a.x_head, a.gate_token, a.gate_head, a.residual_token, a.residual_head, a.out_token, a.out_head})
        if (stride < 0) return failf("%s: negative stride", who);
    const int64_t size = size_of(a.dtype), out_size = size_of(a.out_dtype), res_size = size_of(a.residual_dtype);
    if (!aligned(a.x, size) || !aligned(a.gate, size) || !aligned(a.out, out_size) || (a.residual != nullptr && !aligned(a.residual, res_size)) ||
        (a.weight != nullptr && !aligned(a.weight, size_of(a.weight_dtype))) || (a.out_dtype == 2 && !aligned(a.scales, 4)))
        return failf("%s: a tensor is misaligned for its type", who);
    gdn::ops::NormParams p{a.x, a.gate, a.weight, a.residual, a.out, a.scales, a.x_token, a.x_head, a.gate_token, a.gate_head,
                           a.residual_token, a.residual_head, a.out_token, a.out_head, a.tokens, a.heads, a.dim,
                           a.dtype, a.weight_dtype, a.residual_dtype, a.out_dtype, a.eps};
    if (gdn::ops::norm_threads(p, 16) > gdn::ops::kMaxNormThreads)
        return failf("%s: rows of %u x %u values are more than one CTA holds", who, a.heads, a.dim);
    const Extent x(a.x, a.x_token, a.x_head, a.tokens, a.heads, a.dim, size), out(a.out, a.out_token, a.out_head, a.tokens, a.heads, a.dim, out_size),
        gate(a.gate, a.gate_token, a.gate_head, a.tokens, a.heads, a.dim, size),
        residual(a.residual, a.residual_token, a.residual_head, a.tokens, a.heads, a.dim, res_size),
        weight(a.weight, 0, 0, 1, 1, a.dim, size_of(a.weight_dtype)), scales(a.out_dtype == 2 ? a.scales : nullptr, 0, 0, 1, 1, a.tokens, 4);
    const bool in_place = a.x == a.out && a.dtype == a.out_dtype && (a.tokens == 1 || a.x_token == a.out_token) &&
                          (a.heads == 1 || a.x_head == a.out_head);
    if (rows_overlap(a.out_token, a.out_head, a.tokens, a.heads, a.dim)) return failf("%s: rows of out overlap", who);
    if (a.residual != nullptr && rows_overlap(a.residual_token, a.residual_head, a.tokens, a.heads, a.dim))
        return failf("%s: rows of the residual overlap", who);
    if (out.meets(gate) || out.meets(residual) || out.meets(weight) || (!in_place && out.meets(x)))
        return failf("%s: out overlaps another tensor", who);
    if (residual.meets(x) || residual.meets(gate) || residual.meets(weight)) return failf("%s: the residual overlaps another tensor", who);
    for (const Extent *e : {&x, &out, &gate, &residual, &weight})
        if (scales.meets(*e)) return failf("%s: scales overlaps another tensor", who);
    return on_device(who, a.device, [&](int sms) { return gdn::ops::launch_norm(p, sms, static_cast<cudaStream_t>(a.stream)); });
}

int gdn_b200_linear(const GdnB200LinearArgs *args) {
    const char *who = "gdn_b200_linear";
    if (args == nullptr) return failf("%s: no arguments", who);
    const GdnB200LinearArgs &a = *args;
    if (a.dtype != 1 && a.dtype != 2) return failf("%s: dtype %d is neither BF16 (1) nor E4M3 (2)", who, a.dtype);
    if (a.bias != nullptr && !float_type(a.bias_dtype)) return failf("%s: bias_dtype %d is neither FP32 (0) nor BF16 (1)", who, a.bias_dtype);
    if (a.residual != nullptr && !float_type(a.residual_dtype))
        return failf("%s: residual_dtype %d is neither FP32 (0) nor BF16 (1)", who, a.residual_dtype);
    if (!float_type(a.out_dtype)) return failf("%s: out_dtype %d is neither FP32 (0) nor BF16 (1)", who, a.out_dtype);
    if (a.activation < 0 || a.activation > 3) return failf("%s: activation %d is not 0 to 3", who, a.activation);
    if (a.tokens == 0 || a.outputs == 0) return 0;
    if (a.inputs == 0) return failf("%s: no inputs", who);
    if (a.tokens > 1u << 24 || a.outputs > 1u << 24 || a.inputs > 1u << 24 || (uint64_t)a.tokens * a.outputs > 1ull << 38)
        return failf("%s: %u x %u x %u is too large", who, a.tokens, a.outputs, a.inputs);
    if (a.x == nullptr || a.weight == nullptr || a.out == nullptr) return failf("%s: x, weight or out is missing", who);
    if (a.dtype == 2 && (a.x_scales == nullptr || a.weight_scales == nullptr)) return failf("%s: 8-bit operands need scales", who);
    const int64_t size = size_of(a.dtype), out_size = size_of(a.out_dtype), res_size = size_of(a.residual_dtype);
    const uint32_t rows = a.activation == 3 ? 2 * a.outputs : a.outputs;
    if (!aligned(a.x, 16) || !aligned(a.weight, 16) || (a.tokens > 1 && a.x_row * size % 16 != 0) || (rows > 1 && a.weight_row * size % 16 != 0))
        return failf("%s: rows of x and weight must start on 16-byte boundaries", who);
    if ((a.tokens > 1 && a.x_row < (int64_t)a.inputs) || (rows > 1 && a.weight_row < (int64_t)a.inputs)) return failf("%s: rows of x or weight overlap", who);
    if (a.tokens > 1 && a.out_row < (int64_t)a.outputs) return failf("%s: rows of out overlap", who);
    if (a.residual != nullptr && a.tokens > 1 && a.residual_row < 0) return failf("%s: negative stride", who);
    if (a.x_row > 1ll << 36 || a.weight_row > 1ll << 36) return failf("%s: rows of x or weight are too far apart", who);
    if (!aligned(a.out, out_size) || (a.residual != nullptr && !aligned(a.residual, res_size)) || (a.bias != nullptr && !aligned(a.bias, size_of(a.bias_dtype))) ||
        (a.dtype == 2 && (!aligned(a.x_scales, 4) || !aligned(a.weight_scales, 4))))
        return failf("%s: a tensor is misaligned for its type", who);
    const Extent out(a.out, a.out_row, 0, a.tokens, 1, a.outputs, out_size), x(a.x, a.x_row, 0, a.tokens, 1, a.inputs, size),
        weight(a.weight, a.weight_row, 0, rows, 1, a.inputs, size), residual(a.residual, a.residual_row, 0, a.tokens, 1, a.outputs, res_size),
        bias(a.bias, 0, 0, 1, 1, rows, size_of(a.bias_dtype)), x_scales(a.dtype == 2 ? a.x_scales : nullptr, 0, 0, 1, 1, a.tokens, 4),
        weight_scales(a.dtype == 2 ? a.weight_scales : nullptr, 0, 0, 1, 1, rows, 4);
    const bool in_place = a.residual == a.out && a.residual_dtype == a.out_dtype && (a.tokens == 1 || a.residual_row == a.out_row);
    if (out.meets(x) || out.meets(weight) || out.meets(bias) || out.meets(x_scales) || out.meets(weight_scales) || (!in_place && out.meets(residual)))
        return failf("%s: out overlaps an input", who);
    const gdn::ops::LinearParams p{a.x, a.weight, a.bias, a.residual, a.x_scales, a.weight_scales, a.out, a.x_row, a.weight_row,
                                   a.residual_row, a.out_row, a.tokens, a.inputs, a.outputs, a.dtype, a.bias_dtype,
                                   a.residual_dtype, a.out_dtype, a.activation, g_drop.exchange(0), g_tiles.exchange(0)};
    return on_device(who, a.device, [&](int sms) {
        auto *launch = p.tiles == 0 && gdn::ops::takes_few(p) ? gdn::ops::launch_linear_few : gdn::ops::launch_linear;
        return launch(p, sms, static_cast<cudaStream_t>(a.stream));
    });
}

int gdn_b200_linear_status(int device) {
    DeviceScope scope(device);
    int status = 0;
    cudaError_t e = scope.error;
    if (e == cudaSuccess) e = cudaDeviceSynchronize(); /* the copy below waits for no stream but its own */
    if (e == cudaSuccess) e = gdn::ops::linear_status(&status);
    if (e != cudaSuccess) return cuda_failf("gdn_b200_linear_status", "cannot read the device", e);
    return status == 0 ? 0 : failf("gdn_b200_linear: a wait on the device ran out; the call's outputs are not valid");
}

int gdn_b200_short_conv(const GdnB200ConvArgs *args) {
    const char *who = "gdn_b200_short_conv";
    if (args == nullptr) return failf("%s: no arguments", who);
    const GdnB200ConvArgs &a = *args;
    if (!float_type(a.dtype)) return failf("%s: dtype %d is neither FP32 (0) nor BF16 (1)", who, a.dtype);
    if (!float_type(a.weight_dtype)) return failf("%s: weight_dtype %d is neither FP32 (0) nor BF16 (1)", who, a.weight_dtype);
    if (a.tail_dtype != 0 && a.tail_dtype != a.dtype) return failf("%s: tail_dtype %d is neither FP32 (0) nor that of x", who, a.tail_dtype);
    if (a.activation != 0 && a.activation != 1) return failf("%s: activation %d is not 0 or 1", who, a.activation);
    if (a.width < 2 || a.width > 4) return failf("%s: width %u is not 2, 3 or 4", who, a.width);
    if (a.tokens > 0x3fffffffu || a.sequences > 0x3fffffu) return failf("%s: %u tokens in %u sequences are too many", who, a.tokens, a.sequences);
    if (a.channels > 1u << 20) return failf("%s: %u channels are too many", who, a.channels);
    if (a.starts == nullptr && a.tokens != a.sequences)
        return failf("%s: without starts every sequence has one token (%u tokens, %u sequences)", who, a.tokens, a.sequences);
    if (a.sequences == 0 && a.tokens != 0) return failf("%s: %u tokens but no sequence", who, a.tokens);
    if (a.sequences == 0 || a.channels == 0) return 0;
    if (a.slots == nullptr && a.tail_slots < a.sequences) return failf("%s: %u slots for %u sequences", who, a.tail_slots, a.sequences);
    if (a.weight == nullptr || (a.tails == nullptr && a.tail_slots != 0)) return failf("%s: weight or tails is missing", who);
    if (a.tokens != 0 && (a.x == nullptr || a.out == nullptr)) return failf("%s: x or out is missing", who);
    if (a.x_token < 0) return failf("%s: negative stride", who);
    if (a.tokens > 1 && a.out_token < (int64_t)a.channels) return failf("%s: rows of out overlap", who);
    if ((a.width > 2 && a.tails_row < (int64_t)a.channels) ||
        (a.tail_slots > 1 && a.tails_slot < (a.width > 2 ? ((int64_t)a.width - 2) * a.tails_row : 0) + (int64_t)a.channels))
        return failf("%s: rows or slots of tails overlap", who);
    const int64_t size = size_of(a.dtype), tail_size = size_of(a.tail_dtype), weight_size = size_of(a.weight_dtype);
    if (!aligned(a.x, size) || !aligned(a.out, size) || !aligned(a.tails, tail_size) || !aligned(a.weight, weight_size) || !aligned(a.bias, weight_size) ||
        !aligned(a.starts, 4) || !aligned(a.slots, 4))
        return failf("%s: a tensor is misaligned for its type", who);
    const Extent x(a.x, a.x_token, 0, a.tokens, 1, a.channels, size), out(a.out, a.out_token, 0, a.tokens, 1, a.channels, size),
        tails(a.tails, a.tails_slot, a.tails_row, a.tail_slots, a.width - 1, a.channels, tail_size),
        weight(a.weight, 0, 0, 1, 1, a.channels * a.width, weight_size), bias(a.bias, 0, 0, 1, 1, a.channels, weight_size);
    if (a.tokens != 0 && (out.meets(x) || out.meets(weight) || out.meets(bias))) return failf("%s: out overlaps an input", who);
    if (a.tail_slots != 0 && (tails.meets(weight) || tails.meets(bias) || (a.tokens != 0 && (tails.meets(x) || tails.meets(out)))))
        return failf("%s: tails overlaps another tensor", who);
    const gdn::ops::ConvParams p{a.x, a.weight, a.bias, a.tails, a.out, a.starts, a.slots, a.fresh, a.x_token, a.out_token, a.tails_slot,
                                 a.tails_row, a.sequences, a.tokens, a.channels, a.width, a.tail_slots, a.dtype, a.weight_dtype,
                                 a.tail_dtype, a.activation};
    return on_device(who, a.device, [&](int sms) { return gdn::ops::launch_conv(p, sms, static_cast<cudaStream_t>(a.stream)); });
}

}  // extern "C"
