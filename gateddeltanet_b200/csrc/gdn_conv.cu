/* gdn_conv.cu -- the short causal convolution over packed sequences, each
 * channel by itself, with the last inputs of every sequence in a pool of slots:
 *   y[t][c] = act(bias[c] + sum_j w[c][j] x[t - (W - 1) + j][c])
 * where what lies before a sequence's first token are the W - 1 rows of its
 * slot (zeros if it is fresh), which then get the sequence's last W - 1 inputs.
 *
 * Bound by HBM: x is read and y written once. A thread takes eight
 * neighbouring channels (or one, where rows are not on 16-byte boundaries)
 * through a tile of tokens, the window and the weights in registers; the loads
 * of the next tokens go out together. The tile in which a sequence begins takes
 * all of its tokens that need its slot's rows, and replaces these after it has
 * read them, so that no other CTA touches them: the new ones are rows of x,
 * which does not change.
 */
#include "gdn_ops.h"
#include "gdn_values.h"

namespace gdn {
namespace ops {

namespace {

constexpr uint32_t kThreads = 128;
constexpr int kAhead = 4; /* tokens whose loads are in flight */

__device__ __forceinline__ uint32_t bound_of(const ConvParams &p, uint32_t n) {
    if (p.starts == nullptr) return n;
    const int32_t s = p.starts[n];
    return s < 0 ? 0u : ((uint32_t)s < p.tokens ? (uint32_t)s : p.tokens);
}

/* The number of entries of starts[0 .. N] that are not above t (for starts that do not decrease). */
__device__ uint32_t begun(const ConvParams &p, uint32_t t) {
    if (p.starts == nullptr) return t + 1 < p.N + 1 ? t + 1 : p.N + 1;
    const uint32_t lane = threadIdx.x & 31;
    uint32_t lo = 0, hi = p.N + 1; /* entries before lo are not above t, those from hi on are */
    while (lo < hi) {
        const uint32_t step = (hi - lo + 31) / 32, i = lo + lane * step;
        const uint32_t below = __popc(__ballot_sync(0xffffffffu, i < hi && bound_of(p, i) <= t));
        if (below == 0) return lo;
        const uint32_t next = lo + (below - 1) * step + 1;
        hi = below < 32 && lo + below * step < hi ? lo + below * step : hi;
        lo = next;
    }
    return lo;
}

/* T: type of x and y. kWide: eight channels a thread. */
template <typename T, bool kWide, int W>
__global__ void __launch_bounds__(kThreads) conv_kernel(const __grid_constant__ ConvParams p, const uint32_t tile) {
    constexpr int C = kWide ? 8 : 1;
    const uint32_t c0 = (blockIdx.y * kThreads + threadIdx.x) * C;
    const bool live = c0 < p.channels;
    const T *x = static_cast<const T *>(p.x) + c0;
    T *y = static_cast<T *>(p.out) + c0;
    auto load = [&](const T *from, float (&v)[C]) {
        if constexpr (kWide)
            load8(from, v);
        else
            v[0] = load1(from);
    };
    auto load_tail = [&](int64_t at, float (&v)[C]) {
        if constexpr (kWide)
            load8(p.tails, at, p.tail_type, v);
        else
            v[0] = load1(p.tails, at, p.tail_type);
    };
    auto store = [&](uint32_t t, const float (&v)[C]) {
        if constexpr (kWide)
            store8(y + t * p.out_token, v);
        else
            store1(y + t * p.out_token, v[0]);
    };
    auto store_tail = [&](int64_t at, const float (&v)[C]) {
        if constexpr (kWide)
            store8(p.tails, at, p.tail_type, v);
        else
            store1(p.tails, at, p.tail_type, v[0]);
    };

    float w[W][C], bias[C];
    if (live) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            bias[c] = p.bias != nullptr ? load1(p.bias, c0 + c, p.weight_type) : 0.0f;
#pragma unroll
            for (int j = 0; j < W; ++j) w[j][c] = load1(p.weight, (int64_t)(c0 + c) * W + j, p.weight_type);
        }
    }
    const uint32_t t0 = blockIdx.x * tile, t1 = min(t0 + tile, p.tokens);
    uint32_t n = t0 < t1 ? begun(p, t0) : 0; /* the sequence of token t0 is n - 1, if it has one */
    uint32_t t = t0;
    float zero[C];
#pragma unroll
    for (int c = 0; c < C; ++c) zero[c] = 0.0f;

    while (t < t1) {
        const uint32_t end = n <= p.N ? bound_of(p, n) : p.tokens; /* the first token of the next sequence */
        if (end <= t && n <= p.N) { /* a sequence without tokens, or starts that decrease */
            ++n;
            continue;
        }
        uint32_t stop = min(end, t1);
        const int64_t slot = n == 0 || n > p.N ? -1 : p.slots == nullptr ? (int64_t)(n - 1) : (int64_t)p.slots[n - 1];
        if (slot < 0 || slot >= (int64_t)p.tail_slots) {
            /* tokens of no sequence, or of one without a slot */
            if (live)
                for (; t < stop; ++t) store(t, zero);
            t = stop;
            ++n;
            continue;
        }
        const uint32_t begin = min(bound_of(p, n - 1), t);
        if (begin < t0) {
            t = max(t, min(end, begin + (W - 1))); /* the tokens before belong to an earlier tile */
            stop = max(stop, t);
        } else {
            stop = min(end, max(t1, begin + (W - 1)));
        }
        const bool fresh = p.fresh != nullptr && p.fresh[n - 1] != 0;
        if (live) {
            /* window: inputs t - (W - 1) .. t - 1 */
            float win[W][C];
            const int64_t rows = slot * p.tails_slot + c0;
            if (t == begin) {
                float old[W][C];
#pragma unroll
                for (int j = 0; j < W - 1; ++j) {
#pragma unroll
                    for (int c = 0; c < C; ++c) old[j][c] = 0.0f;
                    if (!fresh) load_tail(rows + j * p.tails_row, old[j]);
#pragma unroll
                    for (int c = 0; c < C; ++c) win[j][c] = old[j][c];
                }
                const uint32_t len = end - begin;
#pragma unroll
                for (int j = 0; j < W - 1; ++j) {
                    float v[C];
                    if (len + j >= W - 1) {
                        load(x + (begin + len + j - (W - 1)) * p.x_token, v);
                    } else {
#pragma unroll
                        for (int c = 0; c < C; ++c) v[c] = 0.0f;
#pragma unroll
                        for (int i = 0; i < W - 1; ++i)
                            if ((uint32_t)i == len + j) {
#pragma unroll
                                for (int c = 0; c < C; ++c) v[c] = old[i][c];
                            }
                    }
                    store_tail(rows + j * p.tails_row, v);
                }
            } else {
#pragma unroll
                for (int j = 0; j < W - 1; ++j) {
#pragma unroll
                    for (int c = 0; c < C; ++c) win[j][c] = 0.0f;
                    if (t < stop) load(x + (int64_t)(t - (W - 1) + j) * p.x_token, win[j]);
                }
            }
            for (; t < stop; t += kAhead) {
                float in[kAhead][C];
#pragma unroll
                for (int a = 0; a < kAhead; ++a)
                    if (t + a < stop) load(x + (int64_t)(t + a) * p.x_token, in[a]);
#pragma unroll
                for (int a = 0; a < kAhead; ++a)
                    if (t + a < stop) {
                        float out[C];
#pragma unroll
                        for (int c = 0; c < C; ++c) {
                            float s = bias[c];
#pragma unroll
                            for (int j = 0; j < W - 1; ++j) s = fmaf(w[j][c], win[j][c], s);
                            s = fmaf(w[W - 1][c], in[a][c], s);
#pragma unroll
                            for (int j = 0; j < W - 2; ++j) win[j][c] = win[j + 1][c];
                            win[W - 2][c] = in[a][c];
                            out[c] = p.silu ? silu(s) : s;
                        }
                        store(t + a, out);
                    }
            }
        }
        t = stop;
        ++n;
    }
    /* fresh sequences without tokens: nobody else touches their slots */
    if (p.starts != nullptr && p.fresh != nullptr)
        for (uint32_t i = blockIdx.x; i < p.N; i += gridDim.x)
            if (p.fresh[i] != 0 && bound_of(p, i + 1) <= bound_of(p, i)) {
                const int64_t slot = p.slots == nullptr ? (int64_t)i : (int64_t)p.slots[i];
                if (live && slot >= 0 && slot < (int64_t)p.tail_slots)
                    for (int j = 0; j < W - 1; ++j) store_tail(slot * p.tails_slot + j * p.tails_row + c0, zero);
            }
}

template <typename T, bool kWide, int W>
cudaError_t launch_conv_t(const ConvParams &p, int sms, cudaStream_t stream) {
    const uint32_t columns = (p.channels + kThreads * (kWide ? 8 : 1) - 1) / (kThreads * (kWide ? 8 : 1));
    /* long tiles read fewer rows twice, short ones make more CTAs */
    uint32_t tile = 32;
    while (tile > 1 && (uint64_t)((p.tokens + tile - 1) / tile) * columns < 8u * (uint32_t)sms) tile /= 2;
    const uint32_t tiles = p.tokens == 0 ? 1 : (p.tokens + tile - 1) / tile;
    return launch(conv_kernel<T, kWide, W>, dim3(tiles, columns), kThreads, 0, stream, p, tile);
}

template <typename T, bool kWide>
cudaError_t launch_conv_w(const ConvParams &p, int sms, cudaStream_t stream) {
    switch (p.width) {
        case 2: return launch_conv_t<T, kWide, 2>(p, sms, stream);
        case 3: return launch_conv_t<T, kWide, 3>(p, sms, stream);
        default: return launch_conv_t<T, kWide, 4>(p, sms, stream);
    }
}

template <typename T>
cudaError_t launch_conv_x(const ConvParams &p, int sms, cudaStream_t stream) {
    const int64_t x_size = sizeof(T), tail_size = p.tail_type == kBF16 ? 2 : 4;
    const bool wide = p.channels % 8 == 0 && on16(p.x) && on16(p.out) && on16(p.tails) &&
                      (p.tokens <= 1 || (p.x_token * x_size % 16 == 0 && p.out_token * x_size % 16 == 0)) &&
                      (p.tail_slots <= 1 || p.tails_slot * tail_size % 16 == 0) && (p.width <= 2 || p.tails_row * tail_size % 16 == 0);
    return wide ? launch_conv_w<T, true>(p, sms, stream) : launch_conv_w<T, false>(p, sms, stream);
}

}  // namespace

cudaError_t launch_conv(const ConvParams &p, int sms, cudaStream_t stream) {
    return p.type == kBF16 ? launch_conv_x<__nv_bfloat16>(p, sms, stream) : launch_conv_x<float>(p, sms, stream);
}

}  // namespace ops
}  // namespace gdn
