// Linear sequence mixers of a frame classifier on channels-last frames [clips, frames, channels]: the short causal
// convolution and the selective state space scan behind it, over whole recordings and one frame at a time.
#include "common.h"

#include <algorithm>

namespace {
#include "vec_io.h"

constexpr int kThreads = 256;

// ------------------------------------------------------------------------------------------------ causal convolution
// y[t, c] = act(bias[c] + sum_k weight[c, k] x[t - (K-1) + k, c]), x before the first frame from the state.
//
// Bytes bound it: x is read once and y written once.  A lane owns 16 bytes of channels and walks kRows frames with
// the last K-1 inputs in registers, so only the K-1 rows in front of each run are read twice.
struct ConvArgs {
    const float *weight, *bias;          // [channels, K], [channels] or null
    const int64_t *lengths;              // [clips] or null
    int64_t x_clip, x_frame;             // strides of x in elements
    int64_t frames, clips;
    int channels, vectors;               // vectors = 16-byte vectors of a row
    int segments, rows;                  // runs of `rows` frames per clip
    int act, reverse;
    uint32_t blocks_per_clip;
};

template <typename T, int K>
__global__ __launch_bounds__(kThreads) void causal_conv_kernel(const T *x, const T *state_in, T *state_out, T *y,
                                                               ConvArgs a) {
    constexpr int V = kVec<T>, H = K - 1, U = 4;
    const int64_t clip = blockIdx.x / a.blocks_per_clip;
    const int64_t item = static_cast<int64_t>(blockIdx.x % a.blocks_per_clip) * kThreads + threadIdx.x;
    const int segment = static_cast<int>(item / a.vectors);
    if (segment >= a.segments) return;
    const int c0 = static_cast<int>(item - static_cast<int64_t>(segment) * a.vectors) * V;
    const int ne = min(V, a.channels - c0);
    const int64_t length = clamp_length(a.lengths, clip, a.frames);
    // frame t of the processing order is row t, or row length-1-t of a reversed clip
    const T *px = x + clip * a.x_clip + (a.reverse && length > 0 ? (length - 1) * a.x_frame : 0) + c0;
    T *py = y + (clip * a.frames + (a.reverse && length > 0 ? length - 1 : 0)) * a.channels + c0;
    const int64_t sx = a.reverse ? -a.x_frame : a.x_frame, sy = a.reverse ? -a.channels : a.channels;
    const int64_t state_at = clip * H * a.channels + c0;

    float w[V][K], b[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int c = min(c0 + e, a.channels - 1);
#pragma unroll
        for (int k = 0; k < K; ++k) w[e][k] = a.weight[static_cast<int64_t>(c) * K + k];
        b[e] = a.bias ? a.bias[c] : 0.0f;
    }
    const int64_t t0 = static_cast<int64_t>(segment) * a.rows, t1 = min(t0 + a.rows, a.frames);
    float past[H > 0 ? H : 1][V];
    Pack<T, V> old[H > 0 ? H : 1];                               // the state: only the first run of a clip looks at it
#pragma unroll
    for (int i = 0; i < H; ++i) {
#pragma unroll
        for (int e = 0; e < V; ++e) old[i].v[e] = static_cast<T>(0.0f);
        if (segment == 0 && state_in != nullptr)
            old[i] = load_pack<T, V>(state_in + state_at + static_cast<int64_t>(i) * a.channels, ne);
    }
#pragma unroll
    for (int i = 0; i < H; ++i) {
        const int64_t t = t0 - H + i;                            // rows >= H: a later run never reaches the state
        Pack<T, V> p = old[i];
        if (t >= 0 && t < length) p = load_pack<T, V>(px + t * sx, ne);
#pragma unroll
        for (int e = 0; e < V; ++e) past[i][e] = static_cast<float>(p.v[e]);
    }
    if (segment == 0 && state_out != nullptr) {
        // the last H inputs of (state, valid frames), oldest first; read before written, so state_out may be state_in
#pragma unroll
        for (int i = 0; i < H; ++i) {
            const int64_t t = length - H + i;
            Pack<T, V> p;
            if (t >= 0) {
                p = load_pack<T, V>(px + t * sx, ne);
            } else {
                p = old[0];
#pragma unroll
                for (int k = 1; k < H; ++k)
                    if (t + H == k) p = old[k];
            }
            store_pack<T, V>(state_out + state_at + static_cast<int64_t>(i) * a.channels, p, ne);
        }
    }
    for (int64_t t = t0; t < t1; t += U) {
        Pack<T, V> in[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (t + u < min(t1, length)) in[u] = load_pack<T, V>(px + (t + u) * sx, ne);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (t + u >= t1) break;
            Pack<T, V> out;
            if (t + u < length) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float v = static_cast<float>(in[u].v[e]);
                    float s = b[e];
#pragma unroll
                    for (int k = 0; k < H; ++k) s = fmaf(w[e][k], past[k][e], s);
                    s = fmaf(w[e][H], v, s);
#pragma unroll
                    for (int k = 0; k + 1 < H; ++k) past[k][e] = past[k + 1][e];
                    if (H > 0) past[H > 0 ? H - 1 : 0][e] = v;
                    out.v[e] = static_cast<T>(activate(s, a.act));
                }
                store_pack<T, V>(py + (t + u) * sy, out, ne);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) out.v[e] = static_cast<T>(0.0f);
                store_pack<T, V>(y + (clip * a.frames + t + u) * a.channels + c0, out, ne);
            }
        }
    }
}

constexpr int kMaxWidth = 8;

template <typename T>
int launch_conv(int width, unsigned blocks, hipStream_t st, const void *x, const void *si, void *so, void *y,
                const ConvArgs &a) {
    auto go = [&](auto k) {
        causal_conv_kernel<T, decltype(k)::value><<<blocks, kThreads, 0, st>>>(
            static_cast<const T *>(x), static_cast<const T *>(si), static_cast<T *>(so), static_cast<T *>(y), a);
    };
    switch (width) {
        case 1: go(std::integral_constant<int, 1>{}); break;
        case 2: go(std::integral_constant<int, 2>{}); break;
        case 3: go(std::integral_constant<int, 3>{}); break;
        case 4: go(std::integral_constant<int, 4>{}); break;
        case 5: go(std::integral_constant<int, 5>{}); break;
        case 6: go(std::integral_constant<int, 6>{}); break;
        case 7: go(std::integral_constant<int, 7>{}); break;
        default: go(std::integral_constant<int, 8>{}); break;
    }
    SEDMI_CHECK_LAUNCH();
    return SEDMI_OK;
}

// ----------------------------------------------------------------------------------------------------- selective scan
//     d_t = softplus(dt_t + dt_bias)        (or dt_t + dt_bias)
//     h_t[c, n] = exp(d_t[c] A[c, n]) h_{t-1}[c, n] + d_t[c] x_t[c] B_t[g(c), n]
//     y_t[c] = (sum_n C_t[g(c), n] h_t[c, n] + D[c] x_t[c]) * silu(z_t[c])
//
// Four lanes share a channel and hold a quarter of its N states each, in registers, from the first frame to the
// last; a workgroup owns 64 channels of one clip.  Tiles of kTile frames go through LDS: there d and d*x are formed
// once per (frame, channel) instead of once per lane, and the four lanes of a channel read them as broadcasts.
constexpr int kChannels = 64;            // per workgroup
constexpr int kTile = 32;                // frames staged at a time
constexpr int kYStride = kChannels + 16; // the four rows a quad group writes land in different banks

struct ScanArgs {
    const void *x, *dt, *B, *C, *z;
    const float *A, *D, *dt_bias;
    const int64_t *lengths;
    const float *state_in;
    float *state_out;
    void *y;
    int64_t x_clip, x_frame, dt_clip, dt_frame, z_clip, z_frame;
    int64_t b_clip, b_frame, b_group, c_clip, c_frame, c_group;
    int64_t frames;
    int channels, states, groups, per_group;
    int blocks_per_group;                // workgroups side by side over the channels of a group
    int softplus, reverse;
    int splits;                          // runs of the time axis
    int64_t run;                         // frames per run, a multiple of kTile
    float *end_state;                    // [clips][splits - 1][channels][states]: state at the end of a run that began at zero
    float *end_step;                     // [clips][splits - 1][channels]: sum of its step sizes
};

// log(1 + exp(x)) = max(x, 0) + log1p(e), e = exp(-|x|) <= 1, and log1p(e) = 2 atanh(s), s = e / (2 + e) <= 1/3, by its
// series: s^2 <= 1/9, the terms left out are below 2^-26 of the sum.  Step sizes of 1e-3 keep all their bits.
__device__ __forceinline__ float softplus(float x) {
    const float e = __builtin_amdgcn_exp2f(-1.44269504f * fabsf(x));
    const float s = e / (2.0f + e), q = s * s;
    float p = 1.0f / 15.0f;
    p = fmaf(p, q, 1.0f / 13.0f);
    p = fmaf(p, q, 1.0f / 11.0f);
    p = fmaf(p, q, 1.0f / 9.0f);
    p = fmaf(p, q, 1.0f / 7.0f);
    p = fmaf(p, q, 1.0f / 5.0f);
    p = fmaf(p, q, 1.0f / 3.0f);
    const float log1p = 2.0f * fmaf(p * q, s, s);
    return x != x ? x : fmaxf(x, 0.0f) + log1p;
}

// Sum over the four lanes of a quad (DPP quad_perm: no LDS).
__device__ __forceinline__ float quad_sum(float v) {
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, true));
    return v;
}

// A * log2(e), so that exp(d A) is one exp2 of a product; -inf is taken as the lowest finite number, for which a step
// of size zero keeps the state instead of making 0 * inf.
__device__ __forceinline__ float decay_rate(float a) {
    const float r = a * 1.44269504088896341f;
    return r < -3.402823466e38f ? -3.402823466e38f : r;
}

template <typename T, int NP, bool END>
__global__ __launch_bounds__(kThreads) void selective_scan_kernel(ScanArgs a) {
    constexpr int N4 = 4 * NP;                                   // states staged per frame, zero beyond a.states
    constexpr int kB = (kTile * N4 + kThreads - 1) / kThreads;   // of them per thread
    __shared__ float s_step[kTile][kChannels][2];                // d, d * x
    __shared__ __attribute__((aligned(16))) float s_b[kTile][N4], s_c[END ? 1 : kTile][N4];
    __shared__ float s_y[END ? 1 : kTile][kYStride];

    const int tid = threadIdx.x;
    unsigned rest = blockIdx.x;
    const int cb = rest % (a.groups * a.blocks_per_group);
    rest /= a.groups * a.blocks_per_group;
    const int splits = END ? a.splits - 1 : a.splits;
    const int split = rest % splits;
    const int64_t clip = rest / splits;
    const int group = cb / a.blocks_per_group;
    const int first = (cb - group * a.blocks_per_group) * kChannels;         // within the group
    const int c0 = group * a.per_group + first;
    const int width = min(kChannels, a.per_group - first);
    const int64_t length = clamp_length(a.lengths, clip, a.frames);
    const int64_t t0 = split * a.run;
    const int64_t t1 = min(t0 + a.run, length);                  // may lie before t0: nothing to do

    const int64_t turn = a.reverse && length > 0 ? length - 1 : 0;
    const int dir = a.reverse ? -1 : 1;
    // staging: two channels of one row per lane, four rows 8 apart per thread
    const int sc = (tid & 31) * 2, sr = tid >> 5;
    const int sn = min(2, width - sc);
    const T *px = static_cast<const T *>(a.x) + clip * a.x_clip + turn * a.x_frame + c0 + sc;
    const T *pd = static_cast<const T *>(a.dt) + clip * a.dt_clip + turn * a.dt_frame + c0 + sc;
    const T *pz = a.z ? static_cast<const T *>(a.z) + clip * a.z_clip + turn * a.z_frame + c0 + sc : nullptr;
    const T *pb = static_cast<const T *>(a.B) + clip * a.b_clip + turn * a.b_frame + group * a.b_group;
    const T *pc = static_cast<const T *>(a.C) + clip * a.c_clip + turn * a.c_frame + group * a.c_group;
    T *py = static_cast<T *>(a.y) + clip * a.frames * a.channels + c0 + sc;
    float bias[2], skip[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        bias[e] = a.dt_bias && e < sn ? a.dt_bias[c0 + sc + e] : 0.0f;
        skip[e] = !END && a.D && e < sn ? a.D[c0 + sc + e] : 0.0f;
    }

    // compute: channel ch of the workgroup, states q * NP ...
    const int ch = tid >> 2, q = tid & 3;
    const bool live = ch < width;
    float rate[NP], h[NP], total = 0.0f;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int n = q * NP + j;
        rate[j] = live && n < a.states ? decay_rate(a.A[static_cast<int64_t>(c0 + ch) * a.states + n]) : 0.0f;
        h[j] = 0.0f;
    }
    if (!END) {
        if (a.state_in != nullptr) {
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                const int n = q * NP + j;
                if (live && n < a.states) h[j] = a.state_in[(clip * a.channels + c0 + ch) * a.states + n];
            }
        }
        for (int s = 0; s < split; ++s) {                        // the runs before this one, joined
            const int64_t at = (clip * (a.splits - 1) + s) * a.channels + c0 + ch;
            const float d = live ? a.end_step[at] : 0.0f;
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                const int n = q * NP + j;
                const float e = live && n < a.states ? a.end_state[at * a.states + n] : 0.0f;
                h[j] = fmaf(__builtin_amdgcn_exp2f(d * rate[j]), h[j], e);
            }
        }
    }

    Pack<T, 2> rx[4], rd[4], rz[4];
    float rb[kB], rc[kB];
    auto fetch = [&](int64_t t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t r = t + sr + 8 * i;
            const int n = r < t1 ? sn : 0;
            rx[i] = load_pack<T, 2>(px + dir * r * a.x_frame, n);
            rd[i] = load_pack<T, 2>(pd + dir * r * a.dt_frame, n);
            if (!END && pz) rz[i] = load_pack<T, 2>(pz + dir * r * a.z_frame, n);
        }
#pragma unroll
        for (int i = 0; i < kB; ++i) {
            const int at = tid + i * kThreads, r = at / N4, n = at % N4;
            const bool on = r < kTile && t + r < t1 && n < a.states;
            rb[i] = on ? static_cast<float>(pb[dir * (t + r) * a.b_frame + n]) : 0.0f;
            if (!END) rc[i] = on ? static_cast<float>(pc[dir * (t + r) * a.c_frame + n]) : 0.0f;
        }
    };
    if (t0 < t1) fetch(t0);
    for (int64_t t = t0; t < t1; t += kTile) {
        Pack<T, 2> cx[4], cz[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = sr + 8 * i;
            float step[2], in[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float v = static_cast<float>(rd[i].v[e]) + bias[e];
                const bool on = t + r < t1 && e < sn;            // behind the end: a step of zero keeps the state
                step[e] = on ? (a.softplus ? softplus(v) : v) : 0.0f;
                in[e] = on ? step[e] * static_cast<float>(rx[i].v[e]) : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) s_step[r][sc + e][0] = step[e], s_step[r][sc + e][1] = in[e];
            cx[i] = rx[i];
            if (!END) cz[i] = rz[i];
        }
#pragma unroll
        for (int i = 0; i < kB; ++i) {
            const int at = tid + i * kThreads;
            if (kTile * N4 >= kThreads || at < kTile * N4) {
                s_b[at / N4][at % N4] = rb[i];
                if (!END) s_c[at / N4][at % N4] = rc[i];
            }
        }
        __syncthreads();
        if (t + kTile < t1) fetch(t + kTile);
        const int steps = static_cast<int>(min(static_cast<int64_t>(kTile), t1 - t));
        for (int r = 0; r < steps; r += 4) {
            float out[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float d = s_step[r + u][ch][0], v = s_step[r + u][ch][1];
                float y = 0.0f;
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    h[j] = fmaf(__builtin_amdgcn_exp2f(d * rate[j]), h[j], v * s_b[r + u][q * NP + j]);
                    if (!END) y = fmaf(h[j], s_c[r + u][q * NP + j], y);
                }
                if (END) total += d;
                else out[u] = quad_sum(y);
            }
            if (!END) s_y[r + q][ch] = q == 0 ? out[0] : q == 1 ? out[1] : q == 2 ? out[2] : out[3];
        }
        __syncthreads();
        if (!END) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = sr + 8 * i;
                if (t + r >= t1 || sn <= 0) continue;
                Pack<T, 2> out;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float v = fmaf(skip[e], static_cast<float>(cx[i].v[e]), s_y[r][sc + e]);
                    if (pz) v *= silu(static_cast<float>(cz[i].v[e]));
                    out.v[e] = static_cast<T>(v);
                }
                store_pack<T, 2>(py + (turn + dir * (t + r)) * a.channels, out, sn);
            }
        }
    }
    if (END) {
        const int64_t at = (clip * (a.splits - 1) + split) * a.channels + c0 + ch;
        if (live) {
            if (q == 0) a.end_step[at] = total;
#pragma unroll
            for (int j = 0; j < NP; ++j)
                if (q * NP + j < a.states) a.end_state[at * a.states + q * NP + j] = h[j];
        }
        return;
    }
    if (sn > 0) {                                                // frames behind the clip's end
        Pack<T, 2> zero;
        zero.v[0] = zero.v[1] = static_cast<T>(0.0f);
        for (int64_t t = max(t0, length) + sr; t < min(t0 + a.run, a.frames); t += 8)
            store_pack<T, 2>(py + t * a.channels, zero, sn);
    }
    if (a.state_out != nullptr && split == splits - 1 && live) {
#pragma unroll
        for (int j = 0; j < NP; ++j)
            if (q * NP + j < a.states) a.state_out[(clip * a.channels + c0 + ch) * a.states + q * NP + j] = h[j];
    }
}

// One frame: the same formulas, the state read and written once.  Bytes of the state bound it.
template <typename T, int NI>
__global__ __launch_bounds__(kThreads) void selective_step_kernel(ScanArgs a, float *state) {
    const int tid = threadIdx.x, ch = tid >> 2, q = tid & 3;
    const unsigned per_clip = a.groups * a.blocks_per_group;
    const int64_t clip = blockIdx.x / per_clip;
    const int cb = blockIdx.x % per_clip;
    const int group = cb / a.blocks_per_group;
    const int first = (cb - group * a.blocks_per_group) * kChannels;
    if (ch >= min(kChannels, a.per_group - first)) return;       // all four lanes of a channel leave together
    const int c = group * a.per_group + first + ch;
    const T *pb = static_cast<const T *>(a.B) + clip * a.b_clip + group * a.b_group;
    const T *pc = static_cast<const T *>(a.C) + clip * a.c_clip + group * a.c_group;
    const float *pa = a.A + static_cast<int64_t>(c) * a.states;
    float *ps = state + (clip * a.channels + c) * a.states;
    const float x = static_cast<float>(static_cast<const T *>(a.x)[clip * a.x_clip + c]);
    float d = static_cast<float>(static_cast<const T *>(a.dt)[clip * a.dt_clip + c]) + (a.dt_bias ? a.dt_bias[c] : 0.0f);
    Pack<float, 4> hs[NI], as[NI];
    Pack<T, 4> bs[NI], cs[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int n = (i * 4 + q) * 4, ne = max(0, min(4, a.states - n));
        hs[i] = load_pack<float, 4>(ps + n, ne);
        as[i] = load_pack<float, 4>(pa + n, ne);
        bs[i] = load_pack<T, 4>(pb + n, ne);
        cs[i] = load_pack<T, 4>(pc + n, ne);
    }
    if (a.softplus) d = softplus(d);
    const float v = d * x;
    float y = 0.0f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int n = (i * 4 + q) * 4, ne = max(0, min(4, a.states - n));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            hs[i].v[e] = fmaf(__builtin_amdgcn_exp2f(d * decay_rate(as[i].v[e])), hs[i].v[e], v * static_cast<float>(bs[i].v[e]));
            y = e < ne ? fmaf(hs[i].v[e], static_cast<float>(cs[i].v[e]), y) : y;
        }
        if (ne > 0) store_pack<float, 4>(ps + n, hs[i], ne);
    }
    y = quad_sum(y);
    if (q == 0) {
        if (a.D) y = fmaf(a.D[c], x, y);
        if (a.z) y *= silu(static_cast<float>(static_cast<const T *>(a.z)[clip * a.z_clip + c]));
        static_cast<T *>(a.y)[clip * a.channels + c] = static_cast<T>(y);
    }
}

constexpr int kMaxStates = 128;

int64_t scan_blocks(int channels, int groups) {
    return static_cast<int64_t>(groups) * sedmi::ceil_div(channels / groups, kChannels);
}

int64_t scan_run(int64_t frames, int splits) {
    return sedmi::ceil_div(sedmi::ceil_div(std::max<int64_t>(frames, 1), splits), kTile) * kTile;
}

int scan_splits(int64_t clips, int64_t frames, int channels, int groups) {
    const int64_t have = clips * scan_blocks(channels, groups);
    if (have >= 512) return 1;
    const int64_t want = sedmi::ceil_div(1024, std::max<int64_t>(1, have));
    const int64_t splits = std::max<int64_t>(1, std::min<int64_t>({want, frames / 128, 64}));
    return static_cast<int>(sedmi::ceil_div(std::max<int64_t>(frames, 1), scan_run(frames, static_cast<int>(splits))));
}

bool dtype_ok(int dtype) {
    return dtype == SEDMI_DTYPE_F32 || dtype == SEDMI_DTYPE_F16 || dtype == SEDMI_DTYPE_BF16;
}

bool scan_shape_ok(int64_t clips, int64_t frames, int channels, int groups, int states) {
    return clips >= 0 && clips <= (int64_t{1} << 24) && frames >= 0 && frames <= (int64_t{1} << 40) && channels > 0 &&
           channels <= (1 << 24) && groups > 0 && channels % groups == 0 && states > 0 && states <= kMaxStates;
}

int check_scan(const sedmi_scan_args *p, const char *who) {
    SEDMI_REQUIRE(p != nullptr, "%s: null arguments", who);
    SEDMI_REQUIRE(dtype_ok(p->dtype), "%s: unknown dtype %d", who, p->dtype);
    SEDMI_REQUIRE(p->channels > 0 && p->groups > 0 && p->channels % p->groups == 0,
                  "%s: channels (%d) must be a positive multiple of groups (%d)", who, p->channels, p->groups);
    SEDMI_REQUIRE(p->states > 0 && p->states <= kMaxStates, "%s: states (%d) must be 1 .. %d", who, p->states, kMaxStates);
    SEDMI_REQUIRE(scan_shape_ok(p->n_clips, p->frames, p->channels, p->groups, p->states), "%s: bad shape", who);
    return SEDMI_OK;
}

ScanArgs scan_args(const sedmi_scan_args *p) {
    ScanArgs a{};
    a.x = p->x, a.dt = p->dt, a.B = p->B, a.C = p->C, a.z = p->z;
    a.A = p->A, a.D = p->D, a.dt_bias = p->dt_bias;
    a.lengths = p->lengths, a.state_in = p->state_in, a.state_out = p->state_out, a.y = p->y;
    a.x_clip = p->x_stride[0], a.x_frame = p->x_stride[1];
    a.dt_clip = p->dt_stride[0], a.dt_frame = p->dt_stride[1];
    a.z_clip = p->z_stride[0], a.z_frame = p->z_stride[1];
    a.b_clip = p->B_stride[0], a.b_frame = p->B_stride[1], a.b_group = p->B_stride[2];
    a.c_clip = p->C_stride[0], a.c_frame = p->C_stride[1], a.c_group = p->C_stride[2];
    a.frames = p->frames, a.channels = p->channels, a.states = p->states, a.groups = p->groups;
    a.per_group = p->channels / p->groups;
    a.blocks_per_group = static_cast<int>(sedmi::ceil_div(a.per_group, kChannels));
    a.softplus = p->dt_softplus, a.reverse = p->reverse;
    return a;
}

template <typename T, bool END>
void launch_scan(int states, unsigned blocks, hipStream_t st, const ScanArgs &a) {
    if (states <= 4) selective_scan_kernel<T, 1, END><<<blocks, kThreads, 0, st>>>(a);
    else if (states <= 8) selective_scan_kernel<T, 2, END><<<blocks, kThreads, 0, st>>>(a);
    else if (states <= 16) selective_scan_kernel<T, 4, END><<<blocks, kThreads, 0, st>>>(a);
    else if (states <= 32) selective_scan_kernel<T, 8, END><<<blocks, kThreads, 0, st>>>(a);
    else if (states <= 64) selective_scan_kernel<T, 16, END><<<blocks, kThreads, 0, st>>>(a);
    else selective_scan_kernel<T, 32, END><<<blocks, kThreads, 0, st>>>(a);
}

template <typename T>
void launch_step(int states, unsigned blocks, hipStream_t st, const ScanArgs &a, float *state) {
    if (states <= 16) selective_step_kernel<T, 1><<<blocks, kThreads, 0, st>>>(a, state);
    else if (states <= 32) selective_step_kernel<T, 2><<<blocks, kThreads, 0, st>>>(a, state);
    else if (states <= 64) selective_step_kernel<T, 4><<<blocks, kThreads, 0, st>>>(a, state);
    else selective_step_kernel<T, 8><<<blocks, kThreads, 0, st>>>(a, state);
}

bool overlap(const void *p, const void *q, size_t bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(p), y = reinterpret_cast<uintptr_t>(q);
    return p != nullptr && q != nullptr && x < y + bytes && y < x + bytes;
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
    SEDMI_REQUIRE(scan_shape_ok(n_clips, frames, channels, 1, 1), "causal_conv1d: bad shape (clips %lld, frames %lld, channels %d)",
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
    a.frames = frames, a.clips = n_clips, a.channels = channels;
    a.act = activation, a.reverse = reverse != 0;
    a.vectors = static_cast<int>(sedmi::ceil_div(channels, static_cast<int64_t>(16 / es)));
    a.rows = 32;
    const int64_t segments = std::max<int64_t>(1, sedmi::ceil_div(frames, a.rows));      // no frames: the state alone
    const int64_t per_clip = sedmi::ceil_div(segments * a.vectors, kThreads), blocks = per_clip * n_clips;
    SEDMI_REQUIRE(segments < (int64_t{1} << 31) && blocks < (int64_t{1} << 31), "causal_conv1d: too many workgroups (%lld)",
                  static_cast<long long>(blocks));
    a.segments = static_cast<int>(segments), a.blocks_per_clip = static_cast<uint32_t>(per_clip);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const double items = static_cast<double>(n_clips) * frames * channels;
    sedmi::ProfileScope scope("causal_conv_kernel", st, 2.0 * width * items, 2.0 * es * items);
    return with_dtype(dtype, [&](auto t) -> int {
        return launch_conv<decltype(t)>(width, static_cast<unsigned>(blocks), st, x, state_in, state_out, y, a);
    });
}

size_t sedmi_selective_scan_workspace_bytes(int64_t n_clips, int64_t frames, int channels, int groups, int states) {
    if (!scan_shape_ok(n_clips, frames, channels, groups, states)) return 0;
    const int splits = scan_splits(n_clips, frames, channels, groups);
    return static_cast<size_t>(n_clips) * (splits - 1) * channels * (states + 1) * sizeof(float);
}

int sedmi_selective_scan(const sedmi_scan_args *p, void *ws, size_t ws_bytes, void *stream) {
    if (int rc = check_scan(p, "selective_scan")) return rc;
    const size_t state_bytes = static_cast<size_t>(p->n_clips) * p->channels * p->states * sizeof(float);
    SEDMI_REQUIRE(!overlap(p->state_in, p->state_out, state_bytes), "selective_scan: state_in and state_out overlap");
    if (p->n_clips == 0) return SEDMI_OK;
    SEDMI_REQUIRE(p->A != nullptr, "selective_scan: null A");
    SEDMI_REQUIRE(p->frames == 0 || (p->x && p->dt && p->B && p->C && p->y), "selective_scan: null x, dt, B, C or y");
    ScanArgs a = scan_args(p);
    a.splits = scan_splits(p->n_clips, p->frames, p->channels, p->groups);
    a.run = scan_run(p->frames, a.splits);
    const size_t need = sedmi_selective_scan_workspace_bytes(p->n_clips, p->frames, p->channels, p->groups, p->states);
    if (need > 0 && (ws == nullptr || ws_bytes < need))
        return sedmi::set_error(SEDMI_ENOMEM, "selective_scan: workspace of %zu bytes, %zu needed", ws_bytes, need);
    a.end_state = static_cast<float *>(ws);
    a.end_step = a.end_state + static_cast<size_t>(p->n_clips) * (a.splits - 1) * p->channels * p->states;
    const int64_t blocks = p->n_clips * scan_blocks(p->channels, p->groups);
    SEDMI_REQUIRE(blocks * a.splits < (int64_t{1} << 31), "selective_scan: too many workgroups");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const double items = static_cast<double>(p->n_clips) * p->frames * p->channels;
    const double es = p->dtype == SEDMI_DTYPE_F32 ? 4 : 2;
    return with_dtype(p->dtype, [&](auto t) -> int {
        using T = decltype(t);
        if (a.splits > 1) {
            sedmi::ProfileScope scope("selective_scan_end_kernel", st, 5 * items * p->states, 2 * es * items);
            launch_scan<T, true>(p->states, static_cast<unsigned>(blocks * (a.splits - 1)), st, a);
        }
        SEDMI_CHECK_LAUNCH();
        {
            sedmi::ProfileScope scope("selective_scan_kernel", st, 7 * items * p->states, (p->z ? 4 : 3) * es * items);
            launch_scan<T, false>(p->states, static_cast<unsigned>(blocks * a.splits), st, a);
        }
        SEDMI_CHECK_LAUNCH();
        return SEDMI_OK;
    });
}

int sedmi_selective_step(const sedmi_scan_args *p, void *stream) {
    if (int rc = check_scan(p, "selective_step")) return rc;
    SEDMI_REQUIRE(p->frames == 1, "selective_step: one frame per clip, not %lld", static_cast<long long>(p->frames));
    SEDMI_REQUIRE(p->lengths == nullptr && p->reverse == 0, "selective_step: lengths and reverse have no meaning here");
    SEDMI_REQUIRE(p->state_in == p->state_out, "selective_step: the state is updated in place (state_in == state_out)");
    if (p->n_clips == 0) return SEDMI_OK;
    SEDMI_REQUIRE(p->A && p->x && p->dt && p->B && p->C && p->y && p->state_out, "selective_step: null pointer");
    const ScanArgs a = scan_args(p);
    const int64_t blocks = p->n_clips * scan_blocks(p->channels, p->groups);
    SEDMI_REQUIRE(blocks < (int64_t{1} << 31), "selective_step: too many workgroups");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const double items = static_cast<double>(p->n_clips) * p->channels;
    sedmi::ProfileScope scope("selective_step_kernel", st, 7 * items * p->states, 8 * items * p->states);
    return with_dtype(p->dtype, [&](auto t) -> int {
        launch_step<decltype(t)>(p->states, static_cast<unsigned>(blocks), st, a, p->state_out);
        SEDMI_CHECK_LAUNCH();
        return SEDMI_OK;
    });
}

}  // extern "C"
