/* gdn_conv.cu -- the short causal convolution over packed sequences, each
 * channel by itself, with the last inputs of every sequence in a pool of slots:
 *   y[t][c] = act(bias[c] + sum_j w[c][j] x[t - (W - 1) + j][c])
 * where what lies before a sequence's first token are the W - 1 rows of its
 * slot (zeros if it is fresh), which then get the sequence's last W - 1 inputs.
 *
 * Bound by HBM: x is read and y written once. A thread takes 16 bytes of
 * neighbouring channels (eight of BF16, four of FP32), or, where rows are not on
 * 16-byte boundaries, two channels as far apart as a CTA has threads, through a
 * tile of tokens, the window in registers and the weights in shared memory; the loads
 * of the next tokens go out together. The tile in which a sequence begins takes
 * all of its tokens that need its slot's rows, and replaces these after it has
 * read them, so that no other CTA touches them: the new ones are rows of x,
 * which does not change.
 *
 * Measured, 6144 channels: 24 prompts of 23982 tokens of BF16 110 us (5.4 TB/s;
 * 108 without silu, 109 with eight tokens of loads on their way through shared
 * memory, so what is left is the reads' and writes' turns), 16000 tokens 74 us,
 * 4096 24.2 to 25.0 (each CTA waits for its weights, the search of starts and x in turn, for 22 tokens), of FP32 37.5 (5.4 TB/s);
 * a token of 64 streams 4.5 to 5.2 us with their tails of FP32 (2.3 TB/s: the launch and two
 * waits for memory, one after the other). Off the boundaries: 4000 tokens of 6145 channels of BF16 34.8 us (2.9
 * TB/s), of 1001 of FP32 11.3 (2.8).
 */
#include "gdn_ops.h"
#include "gdn_values.h"

namespace gdn {
namespace ops {

namespace {

constexpr uint32_t kThreads = 128;
/* Tokens computed together, while the loads of as many more are in flight: with two 64 registers and eight CTAs an SM,
 * with four 90 and five. 24 ragged prompts of BF16 117 us with two, 122 with four; 4 x 1000 tokens of FP32 48.8 and 43.4. */
__host__ __device__ constexpr int ahead_of(int channels) { return channels == 8 ? 2 : 4; }
__host__ __device__ constexpr int ctas_of(int channels) { return channels == 4 ? 5 : 8; }
constexpr uint32_t kMaxTile = 128; /* tokens of a CTA */

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

/* A thread's channels: C neighbours (16 bytes), or, where rows are not on 16-byte boundaries, two that are `gap`
 * apart (0: the second is past the end, and follows the first one's values without being stored). */
template <typename T, bool kWide>
struct Lane {
    static constexpr int C = kWide ? 16 / sizeof(T) : 2;
    uint32_t gap;
    static __device__ __forceinline__ void unpack(const uint4 &w, float (&v)[C]) {
        if constexpr (C == 8)
            unpack8(w, v);
        else if constexpr (C == 4)
            v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
        else
            v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y);
    }
    /* as it is in memory (two channels apart: as FP32) */
    __device__ __forceinline__ uint4 fetch(const T *p) const {
        if constexpr (kWide)
            return __ldcg(reinterpret_cast<const uint4 *>(p));
        else
            return make_uint4(__float_as_uint(load1(p)), __float_as_uint(load1(p + gap)), 0, 0);
    }
    __device__ __forceinline__ void put(T *p, const float (&v)[C]) const {
        if constexpr (C == 8) {
            *reinterpret_cast<uint4 *>(p) = pack8(v);
        } else if constexpr (C == 4) {
            *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            store1(p, v[0]);
            if (gap) store1(p + gap, v[1]);
        }
    }
    __device__ __forceinline__ void get_tail(const ConvParams &p, int64_t at, float (&v)[C]) const {
        if constexpr (C == 8)
            load8(p.tails, at, p.tail_type, v);
        else if constexpr (C == 4) /* x is FP32, and so are the tails */
            unpack(__ldcg(reinterpret_cast<const uint4 *>(static_cast<const float *>(p.tails) + at)), v);
        else
            v[0] = load1(p.tails, at, p.tail_type), v[1] = load1(p.tails, at + gap, p.tail_type);
    }
    __device__ __forceinline__ void put_tail(const ConvParams &p, int64_t at, const float (&v)[C]) const {
        if constexpr (C == 8) {
            store8(p.tails, at, p.tail_type, v);
        } else if constexpr (C == 4) {
            *reinterpret_cast<float4 *>(static_cast<float *>(p.tails) + at) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            store1(p.tails, at, p.tail_type, v[0]);
            if (gap) store1(p.tails, at + gap, p.tail_type, v[1]);
        }
    }
};

/* for results of type T, with the same bits as silu2 */
template <typename T>
__device__ __forceinline__ float silu_of(float x) {
    return sizeof(T) == 4 ? silu(x) : silu_short(x);
}

/* The weights of a CTA's channels in shared memory, by pairs of channels: four taps each, the last one
 * meets the token itself (a shorter width has zeros in front, which nobody reads). One more row than
 * threads, so that threads that fill neighbouring channels use different banks. */
template <int C, uint32_t kLanes, bool kWide>
struct Weights {
    float4 pairs[(C + 1) / 2][2][kLanes + 1]; /* taps 0 and 1 of both channels, taps 2 and 3 */
    __device__ __forceinline__ uint64_t tap(int pair, int j, uint32_t lane) const {
        const float4 e = pairs[pair][j >> 1][lane];
        return j & 1 ? pair_of(e.z, e.w) : pair_of(e.x, e.y);
    }
    /* the four of channel c */
    __device__ __forceinline__ float4 of(int c, uint32_t lane) const {
        const float4 a = pairs[c / 2][0][lane], b = pairs[c / 2][1][lane];
        return c & 1 ? make_float4(a.y, a.w, b.y, b.w) : make_float4(a.x, a.z, b.x, b.z);
    }
    template <int W>
    __device__ __forceinline__ void fill(const ConvParams &p, uint32_t first) {
        constexpr int kEach = (kLanes * C + kThreads - 1) / kThreads;
        const bool whole = W == 4 && p.weight_type == kF32 && on16(p.weight);
        float v[kEach][4];
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const uint32_t i = k * kThreads + threadIdx.x, c = first + i;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[k][j] = 0.0f;
            if (i >= kLanes * C || c >= p.channels) continue;
            if (whole) {
                const float4 e = *reinterpret_cast<const float4 *>(static_cast<const float *>(p.weight) + (size_t)c * 4);
                v[k][0] = e.x, v[k][1] = e.y, v[k][2] = e.z, v[k][3] = e.w;
            } else {
#pragma unroll
                for (int j = 0; j < W; ++j) v[k][4 - W + j] = load1(p.weight, (int64_t)c * W + j, p.weight_type);
            }
        }
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const uint32_t i = k * kThreads + threadIdx.x, of = kWide ? i % C : i / kLanes, lane = kWide ? i / C : i % kLanes;
            if (i < kLanes * C) {
#pragma unroll
                for (int j = 0; j < 4; ++j) reinterpret_cast<float *>(&pairs[of / 2][j >> 1][lane])[(j & 1) * 2 + (of & 1)] = v[k][j];
            }
        }
    }
};

/* bias + sum of weights times the window's values (oldest first) and the token's own, in this order */
template <int W>
__device__ __forceinline__ float tap(const float4 &w, float bias, const float (&v)[W]) {
    float s = bias;
    if constexpr (W > 3) s = fmaf(w.x, v[W - 4], s);
    if constexpr (W > 2) s = fmaf(w.y, v[W - 3], s);
    s = fmaf(w.z, v[W - 2], s);
    return fmaf(w.w, v[W - 1], s);
}

/* T: type of x and y. kWide: 16 bytes of channels a thread. */
template <typename T, bool kWide, int W>
__global__ void __launch_bounds__(kThreads, ctas_of(Lane<T, kWide>::C)) conv_kernel(const __grid_constant__ ConvParams p, const uint32_t tile) {
    using L = Lane<T, kWide>;
    constexpr int C = L::C, kAhead = ahead_of(C);
    __shared__ Weights<C, kThreads, kWide> weights;
    /* the columns of a tile next to one another: their rows are */
    const uint32_t columns = (p.channels + kThreads * C - 1) / (kThreads * C), row = blockIdx.x / columns, column = blockIdx.x - row * columns;
    const uint32_t tid = threadIdx.x, c0 = kWide ? (column * kThreads + tid) * C : column * kThreads * C + tid;
    const bool live = c0 < p.channels;
    const L at{c0 + kThreads < p.channels ? kThreads : 0};
    const T *x = static_cast<const T *>(p.x) + c0;
    T *y = static_cast<T *>(p.out) + c0;
    wait_for_previous();
    weights.template fill<W>(p, column * kThreads * C);
    float bias[C];
#pragma unroll
    for (int c = 0; c < C; ++c) bias[c] = live && p.bias != nullptr ? load1(p.bias, c0 + (kWide ? c : c * at.gap), p.weight_type) : 0.0f;
    __syncthreads();
    const uint32_t t0 = row * tile, t1 = min(t0 + tile, p.tokens);
    uint32_t n = t0 < t1 ? begun(p, t0) : 0; /* the sequence of token t0 is n - 1, if it has one */
    uint32_t t = t0;
    float zero[C];
#pragma unroll
    for (int c = 0; c < C; ++c) zero[c] = 0.0f;

    while (t < t1) {
        const uint32_t end = n <= p.N ? bound_of(p, n) : p.tokens; /* the first token of the next sequence */
        if (end <= t && n <= p.N) { /* a sequence without tokens, of which there may be many, or starts that decrease */
            n = max(n + 1, begun(p, t));
            continue;
        }
        const int64_t slot = n == 0 || n > p.N ? -1 : p.slots == nullptr ? (int64_t)(n - 1) : (int64_t)p.slots[n - 1];
        if (slot < 0 || slot >= (int64_t)p.tail_slots) {
            /* tokens of no sequence, or of one without a slot */
            const uint32_t stop = min(end, t1);
            if (live)
                for (; t < stop; ++t) at.put(y + t * p.out_token, zero);
            t = stop;
            ++n;
            continue;
        }
        const ConvPart part = conv_part(bound_of(p, n - 1), end, t, t0, t1, W - 1);
        const uint32_t stop = part.stop;
        t = part.t;
        if (live) {
            if (part.begins) {
                /* the tokens that meet the slot's rows, one by one */
                const bool fresh = p.fresh != nullptr && p.fresh[n - 1] != 0;
                const int64_t rows = slot * p.tails_slot + c0;
                const uint32_t few = min((uint32_t)(W - 1), end - t);
                float win[W - 1][C];
#pragma unroll
                for (int j = 0; j < W - 1; ++j) {
#pragma unroll
                    for (int c = 0; c < C; ++c) win[j][c] = 0.0f;
                    if (!fresh) at.get_tail(p, rows + j * p.tails_row, win[j]);
                }
                for (uint32_t i = 0; i < few; ++i) {
                    float in[C], out[C];
                    L::unpack(at.fetch(x + (int64_t)(t + i) * p.x_token), in);
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        float v[W];
#pragma unroll
                        for (int j = 0; j < W - 1; ++j) v[j] = win[j][c];
                        v[W - 1] = in[c];
                        const float s = tap<W>(weights.of(c, tid), bias[c], v);
                        out[c] = p.silu ? silu_of<T>(s) : s;
#pragma unroll
                        for (int j = 0; j < W - 1; ++j) win[j][c] = v[j + 1];
                    }
                    at.put(y + (int64_t)(t + i) * p.out_token, out);
                }
                /* the window is now the slot's new content, unless there are more tokens */
                const bool more = end - t > W - 1;
#pragma unroll
                for (int j = 0; j < W - 1; ++j) {
                    if (more) L::unpack(at.fetch(x + ((int64_t)end - (W - 1) + j) * p.x_token), win[j]);
                    at.put_tail(p, rows + j * p.tails_row, win[j]);
                }
                t += few;
            }
            /* the others, kAhead at a time, whose W - 1 inputs before them are in x */
            uint4 in[W - 1 + kAhead], next[kAhead];
            if (t < stop) {
#pragma unroll
                for (int j = 0; j < W - 1; ++j) in[j] = at.fetch(x + ((int64_t)t - (W - 1) + j) * p.x_token);
#pragma unroll
                for (int a = 0; a < kAhead; ++a) next[a] = at.fetch(x + (int64_t)min(t + a, stop - 1) * p.x_token);
            }
            for (; t < stop; t += kAhead) {
#pragma unroll
                for (int a = 0; a < kAhead; ++a) in[W - 1 + a] = next[a];
                if (t + kAhead < stop) {
#pragma unroll
                    for (int a = 0; a < kAhead; ++a) next[a] = at.fetch(x + (int64_t)min(t + kAhead + a, stop - 1) * p.x_token);
                }
                uint32_t result[kAhead][4];
                auto word = [](const uint4 &v, int q) { return q == 0 ? v.x : q == 1 ? v.y : q == 2 ? v.z : v.w; };
                /* two channels at a time: a word of 16-bit inputs, two of 32 bits */
#pragma unroll
                for (int q = 0; q < C / 2; ++q) {
                    uint64_t v[W - 1 + kAhead], w[W];
#pragma unroll
                    for (int j = 0; j < W; ++j) w[j] = weights.tap(q, 4 - W + j, tid);
#pragma unroll
                    for (int j = 0; j < W - 1 + kAhead; ++j)
                        v[j] = C == 8 ? pair_of(low_bf16(word(in[j], q)), high_bf16(word(in[j], q)))
                                      : pair_of(__uint_as_float(word(in[j], 2 * q)), __uint_as_float(word(in[j], 2 * q + 1)));
                    const uint64_t b = pair_of(bias[2 * q], bias[2 * q + 1]);
#pragma unroll
                    for (int a = 0; a < kAhead; ++a) {
                        uint64_t o = b;
#pragma unroll
                        for (int j = 0; j < W; ++j) o = fma2(w[j], v[a + j], o);
                        if (p.silu) o = silu2<sizeof(T) == 4>(o);
                        float lo, hi;
                        split(o, lo, hi);
                        if (C == 8)
                            result[a][q] = pack_bf16(lo, hi);
                        else
                            result[a][2 * q] = __float_as_uint(lo), result[a][2 * q + 1] = __float_as_uint(hi);
                    }
                }
#pragma unroll
                for (int a = 0; a < kAhead; ++a)
                    if (t + a < stop) {
                        T *to = y + (int64_t)(t + a) * p.out_token;
                        if constexpr (kWide)
                            *reinterpret_cast<uint4 *>(to) = make_uint4(result[a][0], result[a][1], result[a][2], result[a][3]);
                        else
                            at.put(to, {__uint_as_float(result[a][0]), __uint_as_float(result[a][1])});
                    }
#pragma unroll
                for (int j = 0; j < W - 1; ++j) in[j] = in[kAhead + j];
            }
        }
        t = stop;
        ++n;
    }
    /* fresh sequences without tokens: nobody else touches their slots */
    if (p.starts != nullptr && p.fresh != nullptr)
        for (uint32_t i = row; i < p.N; i += gridDim.x / columns)
            if (p.fresh[i] != 0 && bound_of(p, i + 1) <= bound_of(p, i)) {
                const int64_t slot = p.slots == nullptr ? (int64_t)i : (int64_t)p.slots[i];
                if (live && slot >= 0 && slot < (int64_t)p.tail_slots)
                    for (int j = 0; j < W - 1; ++j) at.put_tail(p, slot * p.tails_slot + j * p.tails_row + c0, zero);
            }
}

/* One token of every sequence (starts null): a warp a token, so that the slots' rows, which are most of
 * what moves, are all under way at once. */
template <typename T, bool kWide, int W>
__global__ void __launch_bounds__(kThreads) conv_step_kernel(const __grid_constant__ ConvParams p) {
    using L = Lane<T, kWide>;
    constexpr int C = L::C;
    __shared__ Weights<C, 32, kWide> weights;
    const uint32_t lane = threadIdx.x & 31, t = blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
    const uint32_t c0 = kWide ? (blockIdx.y * 32 + lane) * C : blockIdx.y * 32 * C + lane;
    const bool live = c0 < p.channels && t < p.tokens;
    const L at{c0 + 32 < p.channels ? 32u : 0u};
    wait_for_previous();
    let_next_start();
    int64_t slot = -1;
    bool fresh = false;
    if (t < p.tokens) {
        slot = p.slots == nullptr ? (int64_t)t : (int64_t)p.slots[t];
        fresh = p.fresh != nullptr && p.fresh[t] != 0;
    }
    const bool known = slot >= 0 && slot < (int64_t)p.tail_slots;
    const int64_t rows = slot * p.tails_slot + c0;
    float win[W][C], out[C], bias[C];
    if (live) L::unpack(at.fetch(static_cast<const T *>(p.x) + t * p.x_token + c0), win[W - 1]);
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
#pragma unroll
        for (int c = 0; c < C; ++c) win[j][c] = 0.0f;
        if (live && known && !fresh) at.get_tail(p, rows + j * p.tails_row, win[j]);
    }
    weights.template fill<W>(p, blockIdx.y * 32 * C);
#pragma unroll
    for (int c = 0; c < C; ++c) bias[c] = live && p.bias != nullptr ? load1(p.bias, c0 + (kWide ? c : c * at.gap), p.weight_type) : 0.0f;
    __syncthreads();
    if (!live) return;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        float v[W];
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = win[j][c];
        const float s = tap<W>(weights.of(c, lane), bias[c], v);
        out[c] = !known ? 0.0f : p.silu ? silu_of<T>(s) : s;
    }
    at.put(static_cast<T *>(p.out) + t * p.out_token + c0, out);
    if (known) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j) at.put_tail(p, rows + j * p.tails_row, win[j + 1]);
    }
}

template <typename T, bool kWide, int W>
cudaError_t launch_conv_t(const ConvParams &p, int sms, cudaStream_t stream) {
    constexpr uint32_t C = Lane<T, kWide>::C;
    if (p.starts == nullptr) {
        const uint32_t columns = (p.channels + 32 * C - 1) / (32 * C);
        return launch_overlapped(conv_step_kernel<T, kWide, W>, dim3((p.tokens + kThreads / 32 - 1) / (kThreads / 32), columns), kThreads, 0, stream, p);
    }
    const uint32_t columns = (p.channels + kThreads * C - 1) / (kThreads * C);
    /* Tiles as short as lets all CTAs run at once (of more than kMaxTile tokens, two or more times all): a tile reads
     * W - 1 rows twice, but one CTA too many costs as long as all of them. 6144 channels of BF16, us with tiles of 24,
     * 32, 48, 64 and 96: 4096 tokens (21 is the shortest) 25.3, 27.5, 30.5, 34.3, 43.1; 16000 (82) 79.4, 78.6, 78.0,
     * 85.5, 76.6. */
    const uint32_t at_once = (uint32_t)(ctas_of(C) * sms) / columns > 0 ? (uint32_t)(ctas_of(C) * sms) / columns : 1;
    const uint32_t times = (uint32_t)(((uint64_t)p.tokens + (uint64_t)at_once * kMaxTile - 1) / ((uint64_t)at_once * kMaxTile));
    uint32_t tile = times == 0 ? 1 : (uint32_t)(((uint64_t)p.tokens + (uint64_t)at_once * times - 1) / ((uint64_t)at_once * times));
    if (tile > 1) tile += tile & 1; /* two tokens at a time */
    const uint32_t tiles = p.tokens == 0 ? 1 : (p.tokens + tile - 1) / tile;
    if ((uint64_t)tiles * columns > 0x7fffffffu) return cudaErrorInvalidConfiguration;
    return launch_overlapped(conv_kernel<T, kWide, W>, dim3(tiles * columns), kThreads, 0, stream, p, tile);
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
    const bool wide = p.channels % (16 / x_size) == 0 && on16(p.x) && on16(p.out) && on16(p.tails) &&
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
