// Short causal depthwise convolution over channels-last frames [clips, frames, channels], over whole recordings and, with
// the last inputs kept as a state, one frame at a time:
//
//     y[t, c] = act(bias[c] + sum_k weight[c, k] x[t - (K-1) + k, c])
//
// Bytes bound it: x is read once and y written once.  A lane owns 16 bytes of channels and walks a run of frames with the
// K inputs it needs in registers, as the words they are in memory, so only the K-1 rows in front of a run are read twice;
// the next four rows are under way while four are summed.  128 x 250 x 2048 bf16, K = 4: 55 us, 4.7 TB/s (a copy: 5.1);
// one frame of 256 x 2048: 4.8 us.
#include "common.h"

#include <algorithm>
#include <type_traits>

namespace {
#include "vec_io.h"

constexpr int kThreads = 256;
constexpr int kMaxWidth = 8;

struct ConvArgs {
    const float *weight, *bias;          // [channels, K], [channels] or null
    const int64_t *lengths;              // [clips] or null
    int64_t x_clip, x_frame;             // strides of x in elements
    int64_t frames;
    int channels, vectors;               // vectors = 16-byte vectors of a row
    int segments, rows;                  // runs of `rows` frames per clip
    int act, reverse;
    int in_place;                        // the states are one buffer
    uint32_t blocks_per_clip;
};

// One lane's run.  FULL: all V channels exist; ACT: the activation.
template <typename T, int K, bool FULL, int ACT>
__device__ __forceinline__ void conv_run(const T *x, const T *state_in, T *state_out, T *y, const ConvArgs &a, int64_t clip,
                                         int segment, int c0, int64_t length) {
    constexpr int V = kVec<T>, H = K - 1, U = 4, P = Pack<T, V>::kPer;
    const int ne = FULL ? V : a.channels - c0;
    auto load = [&](const T *p) { return load_pack<T, V>(p, FULL ? V : ne); };
    auto store = [&](T *p, const Pack<T, V> &v) { stream_pack<T, V>(p, v, FULL ? V : ne); };
    // frame t of the processing order is row t, or row length - 1 - t of a reversed clip
    const int64_t turn = a.reverse && length > 0 ? length - 1 : 0;
    const int64_t sx = a.reverse ? -a.x_frame : a.x_frame, sy = a.reverse ? -a.channels : a.channels;
    const T *px = x + clip * a.x_clip + turn * a.x_frame + c0;
    T *py = y + (clip * a.frames + turn) * a.channels + c0;
    const int64_t state_at = clip * H * a.channels + c0;
    const int64_t t0 = static_cast<int64_t>(segment) * a.rows, t1 = min(t0 + a.rows, a.frames), tv = min(t1, length);

    Pack<T, V> win[H + U], next[U];                              // H past inputs, then U new ones
#pragma unroll
    for (int i = 0; i < H; ++i) {
        const int64_t t = t0 - H + i;                            // rows >= H: only the first run looks at the state
        win[i] = Pack<T, V>::zero();
        if (t >= 0 && t < length) win[i] = load(px + t * sx);
        if (t < 0 && state_in != nullptr) win[i] = load(state_in + state_at + static_cast<int64_t>(i) * a.channels);
    }
    const T *pn = px + t0 * sx;                                  // the next row to load
    auto fetch = [&]() {
#pragma unroll
        for (int u = 0; u < U; ++u) next[u] = load(pn + u * sx);
        pn += U * sx;
    };
    int64_t rows = tv - t0;                                      // valid frames of this run, <= 0: none
    if (rows >= U) fetch();

    // the V x K weights of these channels are adjacent
    float w[V * K], b[V];
    if constexpr (FULL) {
#pragma unroll
        for (int i = 0; i < V * K / 4; ++i) {
            const auto p = *reinterpret_cast<const Pack<float, 4> *>(a.weight + static_cast<int64_t>(c0) * K + 4 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[4 * i + e] = p.get(e);
        }
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const auto p = a.bias ? *reinterpret_cast<const Pack<float, 4> *>(a.bias + c0 + 4 * i) : Pack<float, 4>::zero();
#pragma unroll
            for (int e = 0; e < 4; ++e) b[4 * i + e] = p.get(e);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V * K; ++i) w[i] = a.weight[static_cast<int64_t>(c0) * K + min(i, ne * K - 1)];
#pragma unroll
        for (int e = 0; e < V; ++e) b[e] = a.bias ? a.bias[c0 + min(e, ne - 1)] : 0.0f;
    }

    if (H > 0 && segment == 0 && state_out != nullptr) {
        // the last H inputs of (state, valid frames), oldest first; this lane alone looks at its channels of the state
        // and has read them, so state_out may be state_in
        Pack<T, V> last[H > 0 ? H : 1];
#pragma unroll
        for (int i = 0; i < H; ++i) {
            const int64_t t = length - H + i;
            last[i] = win[0];
#pragma unroll
            for (int k = 1; k < H; ++k)
                if (t + H == k) last[i] = win[k];
            if (t >= 0) last[i] = load(px + t * sx);
        }
#pragma unroll
        for (int i = 0; i < H; ++i)
            store_pack<T, V>(state_out + state_at + static_cast<int64_t>(i) * a.channels, last[i], FULL ? V : ne);
    }

    T *to = py + t0 * sy;
    auto sum = [&](auto count) {                                 // of the first `count` new rows; then the window moves on
        constexpr int N = decltype(count)::value;
        Pack<T, V> out[N];
#pragma unroll
        for (int i = 0; i < V / P; ++i) {                        // a word of channels at a time
            float s[N][P];
#pragma unroll
            for (int e = 0; e < P; ++e) {
                float f[H + N];
#pragma unroll
                for (int r = 0; r < H + N; ++r) f[r] = win[r].get(i * P + e);
#pragma unroll
                for (int u = 0; u < N; ++u) {
                    float v = b[i * P + e];
#pragma unroll
                    for (int k = 0; k < K; ++k) v = fmaf(w[(i * P + e) * K + k], f[u + k], v);
                    s[u][e] = activate<ACT>(v);
                }
            }
#pragma unroll
            for (int u = 0; u < N; ++u) out[u].set_word(i, s[u]);
        }
#pragma unroll
        for (int u = 0; u < N; ++u) store(to + u * sy, out[u]);
        to += N * sy;
#pragma unroll
        for (int i = 0; i < H; ++i) win[i] = win[N + i];
    };
    for (; rows >= U; rows -= U) {
#pragma unroll
        for (int u = 0; u < U; ++u) win[H + u] = next[u];
        if (rows >= 2 * U) fetch();
        sum(std::integral_constant<int, U>{});
    }
    for (; rows > 0; --rows) {
        win[H] = load(pn);
        pn += sx;
        sum(std::integral_constant<int, 1>{});
    }
    for (int64_t t = max(t0, length); t < t1; ++t)
        store(y + (clip * a.frames + t) * a.channels + c0, Pack<T, V>::zero());
}

template <typename T, int K, int ACT>
__global__ __launch_bounds__(kThreads) void causal_conv_kernel(const T *x, const T *state_in, T *state_out, T *y,
                                                               ConvArgs a) {
    constexpr int V = kVec<T>;
    const int64_t clip = blockIdx.x / a.blocks_per_clip;
    const int64_t item = static_cast<int64_t>(blockIdx.x % a.blocks_per_clip) * kThreads + threadIdx.x;
    const int segment = static_cast<int>(item / a.vectors);
    if (segment >= a.segments) return;
    int c0 = static_cast<int>(item - static_cast<int64_t>(segment) * a.vectors) * V;
    const int64_t length = clamp_length(a.lengths, clip, a.frames);
    // The last vector of a row that is no whole number of them moves back over its neighbour's channels: both lanes write
    // the same values there (16 x 1000 x 2047 f16 46 us, 50 with the lane's own body for single channels).  Not where the
    // state changes under the neighbour's reads.
    if (c0 + V > a.channels && a.channels >= V && !a.in_place) c0 = a.channels - V;
    if (c0 + V <= a.channels) conv_run<T, K, true, ACT>(x, state_in, state_out, y, a, clip, segment, c0, length);
    else conv_run<T, K, false, ACT>(x, state_in, state_out, y, a, clip, segment, c0, length);
}

template <typename T, int K>
void launch_conv(unsigned blocks, hipStream_t st, const T *x, const T *si, T *so, T *y, const ConvArgs &a) {
    with_activation(a.act, [&](auto act) {
        causal_conv_kernel<T, K, decltype(act)::value><<<blocks, kThreads, 0, st>>>(x, si, so, y, a);
    });
}

template <typename T>
void launch_conv(int width, unsigned blocks, hipStream_t st, const T *x, const T *si, T *so, T *y, const ConvArgs &a) {
    switch (width) {
        case 1: launch_conv<T, 1>(blocks, st, x, si, so, y, a); break;
        case 2: launch_conv<T, 2>(blocks, st, x, si, so, y, a); break;
        case 3: launch_conv<T, 3>(blocks, st, x, si, so, y, a); break;
        case 4: launch_conv<T, 4>(blocks, st, x, si, so, y, a); break;
        case 5: launch_conv<T, 5>(blocks, st, x, si, so, y, a); break;
        case 6: launch_conv<T, 6>(blocks, st, x, si, so, y, a); break;
        case 7: launch_conv<T, 7>(blocks, st, x, si, so, y, a); break;
        default: launch_conv<T, 8>(blocks, st, x, si, so, y, a); break;
    }
}

}  // namespace

extern "C" {

int sedmi_causal_conv1d(const void *x, int64_t x_stride_clip, int64_t x_stride_frame, const float *weight,
                        const float *bias, const int64_t *lengths, const void *state_in, void *state_out, void *y,
                        int64_t n_clips, int64_t frames, int channels, int width, int activation, int reverse,
                        int dtype, void *stream) {
    SEDMI_REQUIRE(dtype_ok(dtype), "causal_conv1d: unknown dtype %d", dtype);
    SEDMI_REQUIRE(width >= 1 && width <= kMaxWidth, "causal_conv1d: width (%d) must be 1 .. %d", width, kMaxWidth);
    SEDMI_REQUIRE(activation >= SEDMI_ACT_NONE && activation <= SEDMI_ACT_GELU, "causal_conv1d: unknown activation %d", activation);
    SEDMI_REQUIRE(sequence_shape_ok(n_clips, frames, channels), "causal_conv1d: bad shape (clips %lld, frames %lld, channels %d)",
                  static_cast<long long>(n_clips), static_cast<long long>(frames), channels);
    const size_t es = dtype == SEDMI_DTYPE_F32 ? 4 : 2;
    const size_t state_bytes = static_cast<size_t>(n_clips) * (width - 1) * channels * es;
    SEDMI_REQUIRE(state_in == state_out || !overlap(state_in, state_out, state_bytes),
                  "causal_conv1d: state_in and state_out overlap without being the same buffer");
    if (n_clips == 0) return SEDMI_OK;
    SEDMI_REQUIRE(weight != nullptr && (frames == 0 || (x != nullptr && y != nullptr)), "causal_conv1d: null x, weight or y");
    ConvArgs a{};
    a.weight = weight, a.bias = bias, a.lengths = lengths;
    a.x_clip = x_stride_clip, a.x_frame = x_stride_frame;
    a.frames = frames, a.channels = channels;
    a.act = activation, a.reverse = reverse != 0;
    a.vectors = static_cast<int>(sedmi::ceil_div(channels, static_cast<int64_t>(16 / es)));
    // Runs of 8 frames fill the card with few clips, longer ones read fewer rows twice and set up less often: up to 32
    // frames while there are more than 4 waves per SIMD.  Measured with runs of 8 / 16 / 32 (us): 1 x 250 x 1024 bf16
    // 5.6 / 7.5 / 11.4, 32 x 250 x 1024 11.3 / 10.8 / 15.0, 128 x 250 x 2048 72 / 65 / 61.
    a.rows = 8;
    while (a.rows < 32 && n_clips * sedmi::ceil_div(frames, a.rows) * a.vectors > 262144) a.rows *= 2;
    a.in_place = state_in != nullptr && state_in == state_out;
    const int64_t segments = std::max<int64_t>(1, sedmi::ceil_div(frames, a.rows));      // no frames: the state alone
    const int64_t per_clip = sedmi::ceil_div(segments * a.vectors, kThreads);
    SEDMI_REQUIRE(segments < (int64_t{1} << 31) && launch_ok(per_clip, kThreads), "causal_conv1d: too many workgroups per clip (%lld)",
                  static_cast<long long>(per_clip));
    a.segments = static_cast<int>(segments), a.blocks_per_clip = static_cast<uint32_t>(per_clip);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const double items = static_cast<double>(n_clips) * frames * channels;
    sedmi::ProfileScope scope("causal_conv_kernel", st, 2.0 * width * items, 2.0 * es * items);
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        const int64_t state = static_cast<int64_t>(width - 1) * channels;
        in_launches(n_clips, per_clip, kThreads, [&](int64_t first, int64_t n) {
            a.lengths = lengths ? lengths + first : nullptr;
            launch_conv<T>(width, static_cast<unsigned>(n * per_clip), st, static_cast<const T *>(x) + first * x_stride_clip,
                           state_in ? static_cast<const T *>(state_in) + first * state : nullptr,
                           state_out ? static_cast<T *>(state_out) + first * state : nullptr,
                           static_cast<T *>(y) + first * frames * channels, a);
        });
        SEDMI_CHECK_LAUNCH();
        return SEDMI_OK;
    });
}

}  // extern "C"
