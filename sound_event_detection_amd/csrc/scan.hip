// Selective state space scan over channels-last frames [clips, frames, channels], over whole recordings and one frame at
// a time: the linear recurrence of a frame classifier.
#include "common.h"

#include <algorithm>
#include <type_traits>

namespace {
#include "vec_io.h"

constexpr int kThreads = 256;

// ----------------------------------------------------------------------------------------------------- selective scan
//     d_t = softplus(dt_t + dt_bias)        (or dt_t + dt_bias)
//     h_t[c, n] = exp(d_t[c] A[c, n]) h_{t-1}[c, n] + d_t[c] x_t[c] B_t[g(c), n]
//     y_t[c] = (sum_n C_t[g(c), n] h_t[c, n] + D[c] x_t[c]) * silu(z_t[c])
//
// Four lanes share a channel and hold a quarter of its N states each, in registers, from the first frame to the
// last; a workgroup owns 64 (or 16) channels of one clip.  Tiles of kTile frames go through LDS: there d and d*x are formed
// once per (frame, channel) instead of once per lane, and the four lanes of a channel read them as broadcasts.
//
// The vector unit bounds it: per (frame, channel, state) one exponential (two issues of four cycles), two products and a
// sum, and 41 operations per (frame, channel) around them: unpacking, softplus, the sums over the quarters, the gate.
// 64 x 250 x 1024 x 16 bf16: 72 - 75 us (135 MB, 26 us at the rate of a copy); the counters give 36.3 million issues, 61 us,
// of which the recurrence has 20.5 million, the exponentials alone 8.2.  2 x 6000 x 1024 x 16 f16 in 32 runs: 101 us, 44 of
// them in the first pass.
constexpr int kTile = 32;                // frames staged at a time
constexpr int kStepChannels = 64;        // per workgroup of the single-frame form

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

// log(1 + exp(x)) = max(x, 0) + log1p(e), e = exp(-|x|) <= 1, and log1p(e) = 2 atanh(s), s = e / (2 + e) <= 1/3:
// atanh(s) = s + s q P(q), q = s^2 <= 1/9, with P the polynomial of degree 3 that is nearest to the series
// 1/3 + q/5 + q^2/7 + ... there (4.5e-9 of the result).  Step sizes of 1e-3 keep all their bits, which a logarithm of
// the rounded sum 1 + e would not give them.  What is lost is the rounding of the exponent's product, |x| 2^-24 of e: the
// result is off by at most 6.1e-7 of itself for x >= -10, 1.0e-6 at -20, 1.9e-6 at -40.
__device__ __forceinline__ float softplus(float x) {
    const float e = __builtin_amdgcn_exp2f(-1.44269504f * fabsf(x));
    const float s = e * __builtin_amdgcn_rcpf(2.0f + e), q = s * s;
    float p = fmaf(0.14005976f, q, 0.14000906f);
    p = fmaf(p, q, 0.20010763f);
    p = fmaf(p, q, 0.33333208f);
    const float half = fmaf(p * q, s, s);
    return fmaf(2.0f, half, fmaxf(x, 0.0f));             // a NaN comes through e
}

// Value of the lane n before this one in its row of 16 (DPP rotation: no LDS).
template <int N>
__device__ __forceinline__ float from_lane_before(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + N, 0xF, 0xF, true));
}

// A * log2(e), so that exp(d A) is one exp2 of a product; -inf is taken as the lowest finite number, for which a step
// of size zero keeps the state instead of making 0 * inf.
__device__ __forceinline__ float decay_rate(float a) {
    const float r = a * 1.44269504088896341f;
    return r < -3.402823466e38f ? -3.402823466e38f : r;
}

// The element behind the first of a pair, moved to its place.
template <typename T>
__device__ __forceinline__ Pack<T, 2> second_first(Pack<T, 2> p, bool move) {
    if constexpr (sizeof(T) == 2) p.w[0] >>= move ? 16 : 0;
    else p.w[0] = move ? p.w[1] : p.w[0];
    return p;
}

using F4 = __attribute__((ext_vector_type(4))) float;

// Lane v of a wave holds channel (v & 3) + 4 (v >> 4) of the wave's 16 and quarter q = (v >> 2) & 3 of its states: with
// NP >= 4 states per lane those are n = 16 k + 4 q + i, k < NP / 4, i < 4.  That is the layout of sixteen 4 x 4 blocks of
// the matrix instruction v_mfma_f32_4x4x1 (row i in register i, column = lane & 3), so d x B^T, an outer product of 4
// channels and 4 states per block, is added to exp(d A) h by the matrix unit while the vector unit, which bounds this
// kernel, forms the next exponents (64 x 250 x 1024 x 16: 83 us without, 77 with, all else equal).  Up to 8 states (NP < 4) a lane holds n = q NP + i and adds them itself.
//
// Two waves per SIMD at least: with at most 256 registers the compiler keeps the matrix instruction's
// accumulators in ordinary registers, which saves eight moves per frame.
//
// WAVES: 4, or 1 for groups of up to 32 channels with up to 16 states, whose workgroups of 64 would leave half of their lanes idle or more.
template <typename T, int NP, bool END, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void selective_scan_kernel(ScanArgs a) {
    constexpr int kThreads = 64 * WAVES, kChannels = 16 * WAVES;
    constexpr int kYStride = kChannels + 16;                     // rows of y that a wave writes together: different banks
    constexpr int N4 = 4 * NP;                                   // states staged per frame, those past a.states copies of the last
    constexpr bool kMatrix = NP >= 4;
    constexpr int kBRows = kThreads / N4 < kTile ? kThreads / N4 : kTile;    // rows of B that the workgroup loads at a time
    constexpr int kB = kTile / kBRows;
    constexpr int kJoin = NP <= 8 ? 8 : 2;                       // runs whose ends are in flight together
    __shared__ float s_step[kTile][kChannels][2];                // d, d * x
    __shared__ __attribute__((aligned(16))) float s_b[kTile][N4], s_c[END ? 1 : kTile][N4];
    __shared__ float s_y[END ? 1 : kTile + 2][kYStride];         // the last two rows: what half of the lanes need not write

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
    const int64_t count = min(t0 + a.run, length) - t0;          // valid frames of this run, <= 0: none

    // staging: two channels of one row per lane, four rows 8 apart per thread.  Of an odd number of channels the last
    // lane loads the pair before it and takes the second; lanes beside the last channel load the last pair for nothing.
    const int64_t turn = a.reverse && length > 0 ? length - 1 : 0;
    const int dir = a.reverse ? -1 : 1;
    const int sc = tid % (kChannels / 2) * 2, sr = tid / (kChannels / 2);
    const int sn = min(2, width - sc), pair = max(0, min(sc, width - 2));
    const bool second = sc - pair == 1 && width > 1;
    const int64_t row0 = turn + dir * t0;
    const int64_t sx = dir * a.x_frame, sd = dir * a.dt_frame, sz = dir * a.z_frame;
    const int64_t sb = dir * a.b_frame, sv = dir * a.c_frame, sy = dir * a.channels;
    const T *px = static_cast<const T *>(a.x) + clip * a.x_clip + row0 * a.x_frame + c0;
    const T *pd = static_cast<const T *>(a.dt) + clip * a.dt_clip + row0 * a.dt_frame + c0;
    const T *pz = static_cast<const T *>(a.z) + (a.z ? clip * a.z_clip + row0 * a.z_frame + c0 : 0);
    const T *pb = static_cast<const T *>(a.B) + clip * a.b_clip + row0 * a.b_frame + group * a.b_group;
    const T *pc = static_cast<const T *>(a.C) + clip * a.c_clip + row0 * a.c_frame + group * a.c_group;
    T *py = static_cast<T *>(a.y) + (clip * a.frames + row0) * a.channels + c0;
    const int64_t ox = sr * sx + pair, od = sr * sd + pair, oz = sr * sz + pair, oy = sr * sy + sc;
    const int br = min(tid / N4, kTile - 1), bn = tid % N4, bl = min(bn, a.states - 1);
    // A state past the last is a copy of it, and C is shared out among the last and its copies in powers of two, exactly: a
    // state of zeros would turn an infinite input into 0 * inf = NaN and pass that on to y.
    const int copies = N4 - a.states, copy = bn - (a.states - 1);
    const float c_share = copy < 0 ? 1.0f : __builtin_amdgcn_ldexpf(1.0f, -min(copy + 1, copies));
    const int64_t ob = br * sb + bl, oc = br * sv + bl;
    const bool gate = !END && a.z != nullptr;
    float bias[2], skip[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int c = c0 + min(sc + e, width - 1);
        bias[e] = a.dt_bias ? a.dt_bias[c] : 0.0f;
        skip[e] = !END && a.D ? a.D[c] : 0.0f;
    }

    // compute: a lane past the last channel repeats it
    const int lane = tid & 63, q = (lane >> 2) & 3;
    const int ch = (tid >> 6) * 16 + (lane >> 4) * 4 + (lane & 3);
    const bool live = ch < width;
    const int cl = c0 + min(ch, width - 1);
    auto state_of = [&](int j) __attribute__((always_inline)) { return kMatrix ? 16 * (j / 4) + 4 * q + j % 4 : q * NP + j; };
    float rate[NP], h[NP], total = 0.0f;
    const float last_rate = decay_rate(a.A[static_cast<int64_t>(cl) * a.states + a.states - 1]);
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const float v = a.A[static_cast<int64_t>(cl) * a.states + min(state_of(j), a.states - 1)];
        rate[j] = state_of(j) < a.states ? decay_rate(v) : last_rate;    // v without the choice: 14 registers more at 64 states
        h[j] = 0.0f;
    }
    if (!END) {
        if (a.state_in != nullptr) {
#pragma unroll
            for (int j = 0; j < NP; ++j) h[j] = a.state_in[(clip * a.channels + cl) * a.states + min(state_of(j), a.states - 1)];
        }
        for (int s = 0; s < split; s += kJoin) {                 // the runs before this one, joined
            float d[kJoin], e[kJoin][NP];
#pragma unroll
            for (int k = 0; k < kJoin; ++k) {
                const int64_t at = (clip * (a.splits - 1) + min(s + k, split - 1)) * a.channels + cl;
                d[k] = a.end_step[at];
#pragma unroll
                for (int j = 0; j < NP; ++j) e[k][j] = a.end_state[at * a.states + min(state_of(j), a.states - 1)];
            }
#pragma unroll
            for (int k = 0; k < kJoin; ++k) {
                if (s + k >= split) break;
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    // half of the run's decay, twice: a growing state's 2^184 has no float32 (it made 0 into NaN), and an
                    // infinite state is not multiplied by zero
                    const float half = __builtin_amdgcn_exp2f(__builtin_amdgcn_fmed3f(0.5f * d[k] * rate[j], -126.0f, 127.0f));
                    h[j] = fmaf(half, half * h[j], e[k][j]);
                }
            }
        }
    }

    Pack<T, 2> rx[4], rd[4], rz[4] = {};
    T rb[kB], rc[kB];
    // The next rows of the run, `left` of them valid; rows past them repeat the last.  kWhole: all kTile are valid;
    // kRows: fewer; kOne: the block has one channel, beside which there may be no memory.
    enum { kWhole, kRows, kOne };
    auto load = [&](auto mode, const T *p, int i, int64_t stride, int64_t at, int left) __attribute__((always_inline)) {
        if constexpr (decltype(mode)::value == kWhole) {
            return load_pack<T, 2>(p + 8 * i * stride + at, 2);
        } else {
            const T *row = p + min(sr + 8 * i, left - 1) * stride;
            if constexpr (decltype(mode)::value == kRows) return load_pack<T, 2>(row + pair, 2);
            else return load_pack<T, 2>(row, 1);
        }
    };
    auto fetch = [&](auto mode, int left) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) rx[i] = load(mode, px, i, sx, ox, left), rd[i] = load(mode, pd, i, sd, od, left);
        if (gate) {
#pragma unroll
            for (int i = 0; i < 4; ++i) rz[i] = load(mode, pz, i, sz, oz, left);
            pz += kTile * sz;
        }
#pragma unroll
        for (int i = 0; i < kB; ++i) {
            if constexpr (decltype(mode)::value == kWhole) {
                rb[i] = pb[i * kBRows * sb + ob];
                if (!END) rc[i] = pc[i * kBRows * sv + oc];
            } else {
                const int r = min(br + i * kBRows, left - 1);
                rb[i] = pb[r * sb + bl];
                if (!END) rc[i] = pc[r * sv + bl];
            }
        }
        px += kTile * sx, pd += kTile * sd, pb += kTile * sb, pc += kTile * sv;
    };
    auto fetch_any = [&](int left) __attribute__((always_inline)) {
        if (left == kTile && width > 1) fetch(std::integral_constant<int, kWhole>{}, kTile);
        else if (width > 1) fetch(std::integral_constant<int, kRows>{}, left);
        else fetch(std::integral_constant<int, kOne>{}, left);
    };
    auto stage = [&](auto whole, auto soft, int left) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = sr + 8 * i;
            rd[i] = second_first(rd[i], second), rx[i] = second_first(rx[i], second);
            float step[2], in[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float v = rd[i].get(e) + bias[e];
                step[e] = decltype(soft)::value ? softplus(v) : v;
                in[e] = step[e] * rx[i].get(e);
                if (!decltype(whole)::value && r >= left) step[e] = in[e] = 0.0f;    // a step of zero keeps the state
            }
            *reinterpret_cast<F4 *>(&s_step[r][sc][0]) = F4{step[0], in[0], step[1], in[1]};
        }
#pragma unroll
        for (int i = 0; i < kB; ++i) {
            const int r = br + i * kBRows;
            const bool on = decltype(whole)::value || r < left;
            if (kB > 1 || tid / N4 < kTile) {
                s_b[r][bn] = on ? static_cast<float>(rb[i]) : 0.0f;
                if (!END) s_c[r][bn] = on ? static_cast<float>(rc[i]) * c_share : 0.0f;
            }
        }
    };
    // sums of y over the quarters for four frames: the lanes 8 apart exchange halves, then those of the odd quarters add
    // their neighbours' and have two frames each
    const bool high = q & 2;
    float *const y_base = &s_y[END ? 0 : (q & 1 ? q - 1 : kTile)][ch];
    const int y_step = q & 1 ? 4 * kYStride : 0;

    auto left_at = [&](int64_t t) __attribute__((always_inline)) { return static_cast<int>(min(static_cast<int64_t>(kTile), count - t)); };
    if (count > 0) fetch_any(left_at(0));
    for (int64_t t = 0; t < count; t += kTile) {
        const int left = left_at(t);
        const bool whole = left == kTile;
        Pack<T, 2> cx[4], cz[4];
        if (whole && a.softplus) stage(std::true_type{}, std::true_type{}, kTile);
        else if (a.softplus) stage(std::false_type{}, std::true_type{}, left);
        else stage(std::false_type{}, std::false_type{}, left);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            cx[i] = a.D ? rx[i] : Pack<T, 2>::zero();            // without D an infinite x must not meet a factor of zero
            cz[i] = second_first(rz[i], second);
        }
        __syncthreads();
        if (t + kTile < count) fetch_any(left_at(t + kTile));
        float *y_at = y_base;
        for (int r = 0; r < left; r += 4) {
            float out[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float d = s_step[r + u][ch][0], v = s_step[r + u][ch][1];
                float y = 0.0f;
                if constexpr (kMatrix) {
#pragma unroll
                    for (int k = 0; k < NP / 4; ++k) {
                        F4 next;
#pragma unroll
                        for (int i = 0; i < 4; ++i) next[i] = __builtin_amdgcn_exp2f(d * rate[4 * k + i]) * h[4 * k + i];
                        next = __builtin_amdgcn_mfma_f32_4x4x1f32(s_b[r + u][16 * k + 4 * q + (lane & 3)], v, next, 0, 0, 0);
                        F4 c;
                        if (!END) c = *reinterpret_cast<const F4 *>(&s_c[r + u][16 * k + 4 * q]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            h[4 * k + i] = next[i];
                            if (!END) y = fmaf(next[i], c[i], y);
                        }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < NP; ++j) {
                        h[j] = fmaf(__builtin_amdgcn_exp2f(d * rate[j]), h[j], v * s_b[r + u][q * NP + j]);
                        if (!END) y = fmaf(h[j], s_c[r + u][q * NP + j], y);
                    }
                }
                if (END) total += d;
                else out[u] = y;
            }
            if (!END) {
                float k0 = high ? out[2] : out[0], k1 = high ? out[3] : out[1];
                k0 += from_lane_before<8>(high ? out[0] : out[2]);
                k1 += from_lane_before<8>(high ? out[1] : out[3]);
                y_at[0] = k0 + from_lane_before<4>(k0);
                y_at[kYStride] = k1 + from_lane_before<4>(k1);
                y_at += y_step;
            }
        }
        __syncthreads();
        if (!END) {
            auto write = [&](auto all, auto gated) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = sr + 8 * i;
                    float v[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        v[e] = fmaf(skip[e], cx[i].get(e), s_y[r][sc + e]);
                        if (decltype(gated)::value) v[e] *= silu(cz[i].get(e));
                    }
                    T *to = py + 8 * i * sy + oy;
                    if constexpr (decltype(all)::value) store_pack<T, 2>(to, Pack<T, 2>::from(v), 2);
                    else if (r < left && sn > 0) store_pack<T, 2>(to, Pack<T, 2>::from(v), sn);
                }
                py += kTile * sy;
            };
            const bool all = whole && width == kChannels;
            if (all && gate) write(std::true_type{}, std::true_type{});
            else if (all) write(std::true_type{}, std::false_type{});
            else if (gate) write(std::false_type{}, std::true_type{});
            else write(std::false_type{}, std::false_type{});
        }
    }
    if (END) {
        const int64_t at = (clip * (a.splits - 1) + split) * a.channels + cl;
        if (live) {
            if (q == 0) a.end_step[at] = total;
#pragma unroll
            for (int j = 0; j < NP; ++j)
                if (state_of(j) < a.states) a.end_state[at * a.states + state_of(j)] = h[j];
        }
        return;
    }
    if (sn > 0) {                                                // frames behind the clip's end
        T *pe = static_cast<T *>(a.y) + clip * a.frames * a.channels + c0 + sc;
        for (int64_t t = max(t0, length) + sr; t < min(t0 + a.run, a.frames); t += 8)
            store_pack<T, 2>(pe + t * a.channels, Pack<T, 2>::zero(), sn);
    }
    if (a.state_out != nullptr && split == splits - 1 && live) {
#pragma unroll
        for (int j = 0; j < NP; ++j)
            if (state_of(j) < a.states) a.state_out[(clip * a.channels + cl) * a.states + state_of(j)] = h[j];
    }
}

// Sum over the four lanes of a quad.
__device__ __forceinline__ float quad_sum(float v) {
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, true));
    return v;
}

// The value of lane I of the quad.
template <int I>
__device__ __forceinline__ float quad_lane(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), I * 0x55, 0xF, 0xF, true));
}

// One frame: the same formulas, the state read and written once; its bytes bound the kernel.  The four lanes of a quad
// share a channel and take 16 bytes of its state in turn, so a quad reads 64 adjacent bytes.  With many streams a quad
// takes the channel of M = 4 of them: their states are in flight together, the decay rates are read once, and each lane
// does the work per channel (step size, gate, output) of one stream.
//
// WHOLE (at least 4 states): every 16-byte piece is loaded whole, the last one moved back over its neighbour's states, and
// lanes past it load it for nothing, so no branch holds up a load (256 streams x 2048 x 16 bf16: 13 us, 5.4 TB/s; 27 with a
// branch for each piece).  Elements in two pieces get the same value from both; every load of a wave comes before its stores.
template <typename T, int NI, int M, bool WHOLE>
__global__ __launch_bounds__(kThreads) void selective_step_kernel(ScanArgs a, float *state, int64_t clips) {
    static_assert(M == 1 || M == 4, "one stream, or one per lane of a quad");
    const int tid = threadIdx.x, ch = tid >> 2, q = tid & 3;
    const unsigned per_clip = a.groups * a.blocks_per_group;
    const int64_t clip0 = blockIdx.x / per_clip * static_cast<int64_t>(M);
    const int cb = blockIdx.x % per_clip;
    const int group = cb / a.blocks_per_group;
    const int first = (cb - group * a.blocks_per_group) * kStepChannels;
    if (ch >= min(kStepChannels, a.per_group - first)) return;       // all four lanes of a channel leave together
    const int c = group * a.per_group + first + ch;
    const float *pa = a.A + static_cast<int64_t>(c) * a.states;
    Pack<float, 4> hs[M][NI], as[NI];
    Pack<T, 4> bs[M][NI], cs[M][NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int n = WHOLE ? min((i * 4 + q) * 4, a.states - 4) : 0, ne = WHOLE ? 4 : a.states;
        if (WHOLE || i * 4 + q == 0) {
            as[i] = load_pack<float, 4>(pa + n, ne);
#pragma unroll
            for (int m = 0; m < M; ++m) {                        // streams past the last repeat it
                const int64_t clip = min(clip0 + m, clips - 1);
                hs[m][i] = load_pack<float, 4>(state + (clip * a.channels + c) * a.states + n, ne);
                bs[m][i] = load_pack<T, 4>(static_cast<const T *>(a.B) + clip * a.b_clip + group * a.b_group + n, ne);
                cs[m][i] = load_pack<T, 4>(static_cast<const T *>(a.C) + clip * a.c_clip + group * a.c_group + n, ne);
            }
        }
    }
    const bool mine = M == 1 ? q == 0 : clip0 + q < clips;       // whether this lane has an output
    const int64_t own = min(clip0 + (M == 1 ? 0 : q), clips - 1);
    const float x = static_cast<float>(static_cast<const T *>(a.x)[own * a.x_clip + c]);
    float d = static_cast<float>(static_cast<const T *>(a.dt)[own * a.dt_clip + c]) + (a.dt_bias ? a.dt_bias[c] : 0.0f);
    const float z = a.z ? static_cast<float>(static_cast<const T *>(a.z)[own * a.z_clip + c]) : 0.0f;
    const float skip = a.D ? a.D[c] : 0.0f;
    if (a.softplus) d = softplus(d);
    const float v = d * x;
    float y = 0.0f;
    auto stream = [&](auto index) __attribute__((always_inline)) {
        constexpr int m = decltype(index)::value;
        const float dm = M == 1 ? d : quad_lane<m>(d), vm = M == 1 ? v : quad_lane<m>(v);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int n0 = (i * 4 + q) * 4, n = WHOLE ? min(n0, a.states - 4) : 0, ne = WHOLE ? 4 : a.states;
            if (n0 >= a.states) continue;
            float h[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                h[e] = fmaf(__builtin_amdgcn_exp2f(dm * decay_rate(as[i].get(e))), hs[m][i].get(e), vm * bs[m][i].get(e));
                sum = e >= n0 - n && e < ne ? fmaf(h[e], cs[m][i].get(e), sum) : sum;
            }
            if (clip0 + m < clips)
                store_pack<float, 4>(state + ((clip0 + m) * a.channels + c) * a.states + n, Pack<float, 4>::from(h), ne);
        }
        sum = quad_sum(sum);
        if (M == 1 || q == m) y = sum;
    };
    stream(std::integral_constant<int, 0>{});
    if constexpr (M == 4) {
        stream(std::integral_constant<int, 1>{});
        stream(std::integral_constant<int, 2>{});
        stream(std::integral_constant<int, 3>{});
    }
    if (!mine) return;
    if (a.D) y = fmaf(skip, x, y);
    if (a.z) y *= silu(z);
    static_cast<T *>(a.y)[own * a.channels + c] = static_cast<T>(y);
}

constexpr int kMaxStates = 128;

int64_t blocks_of(int channels, int groups, int width) {
    return static_cast<int64_t>(groups) * sedmi::ceil_div(channels / groups, width);
}

// Waves of a scan's workgroup, 16 channels each.  Four against one for narrow groups (us): 64 clips x 1165 frames x 29
// channels x 16 states 52.6 / 41.5, 128 x 250 x 4 groups of 16 45.5 / 36.4, 47 x 138 x 4 groups of 5 27.7 / 20.9; with 32
// states, whose rows take a wave alone twice as long to stage, 1 x 74 x 4 groups of 14 20.8 / 22.1.
int scan_waves(int channels, int groups, int states) { return channels / groups <= 32 && states <= 16 ? 1 : 4; }

int64_t scan_run(int64_t frames, int splits) {
    return sedmi::ceil_div(sedmi::ceil_div(std::max<int64_t>(frames, 1), splits), kTile) * kTile;
}

// Runs of the time axis.  Splitting costs a second pass over all but the last run (0.6 of the scan itself), a launch and
// the joining, so time is only split where workgroups are missing, up to four workgroups per compute unit (16 waves).  Runs
// are whole tiles of the same number: one each for a whole number of tiles, two where frames are left over (250 frames: 4
// runs of 64).  Measured, whole against split (N = 16, us): 16 workgroups of 4 waves x 250 frames 30 / 18, 10 x 1000 103 / 22,
// 64 x 250 30 / 19, 32 x 6000 605 / 107; 256 x 250 32 / 39, 384 x 1000 152 / 169; 8 x 64 10 / 12.  More than 64 runs
// lose to the joining (4 x 6000: 64 runs 41, 94 runs 47).
int scan_splits(int64_t clips, int64_t frames, int channels, int groups, int states) {
    const int waves = scan_waves(channels, groups, states);
    const int64_t have = std::max<int64_t>(1, clips * blocks_of(channels, groups, 16 * waves) * waves);
    if (have >= 768 || frames < 128) return 1;
    const int64_t splits = std::min<int64_t>({sedmi::ceil_div(4096, have), frames / kTile, 64});
    return static_cast<int>(sedmi::ceil_div(frames, scan_run(frames, static_cast<int>(splits))));
}

bool scan_shape_ok(int64_t clips, int64_t frames, int channels, int groups, int states) {
    return sequence_shape_ok(clips, frames, channels) && groups > 0 && channels % groups == 0 && states > 0 &&
           states <= kMaxStates;
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
    a.softplus = p->dt_softplus, a.reverse = p->reverse;
    return a;
}

// The arguments for the clips from `first` on.
template <typename T>
ScanArgs scan_args(ScanArgs a, int64_t first) {
    const auto move = [&](const void *&p, int64_t stride) { if (p) p = static_cast<const T *>(p) + first * stride; };
    move(a.x, a.x_clip), move(a.dt, a.dt_clip), move(a.z, a.z_clip), move(a.B, a.b_clip), move(a.C, a.c_clip);
    a.y = static_cast<T *>(a.y) + first * a.frames * a.channels;
    const int64_t state = first * a.channels * a.states;
    if (a.state_in) a.state_in += state;
    if (a.state_out) a.state_out += state;
    if (a.lengths) a.lengths += first;
    return a;
}

template <typename T, bool END>
void launch_scan(int states, int waves, unsigned blocks, hipStream_t st, const ScanArgs &a) {
    if (waves == 1) {
        if (states <= 4) selective_scan_kernel<T, 1, END, 1><<<blocks, 64, 0, st>>>(a);
        else if (states <= 8) selective_scan_kernel<T, 2, END, 1><<<blocks, 64, 0, st>>>(a);
        else selective_scan_kernel<T, 4, END, 1><<<blocks, 64, 0, st>>>(a);
    } else {
        if (states <= 4) selective_scan_kernel<T, 1, END, 4><<<blocks, 256, 0, st>>>(a);
        else if (states <= 8) selective_scan_kernel<T, 2, END, 4><<<blocks, 256, 0, st>>>(a);
        else if (states <= 16) selective_scan_kernel<T, 4, END, 4><<<blocks, 256, 0, st>>>(a);
        else if (states <= 32) selective_scan_kernel<T, 8, END, 4><<<blocks, 256, 0, st>>>(a);
        else if (states <= 64) selective_scan_kernel<T, 16, END, 4><<<blocks, 256, 0, st>>>(a);
        else selective_scan_kernel<T, 32, END, 4><<<blocks, 256, 0, st>>>(a);
    }
}

template <typename T, int M>
void launch_step(int states, unsigned blocks, hipStream_t st, const ScanArgs &a, float *state, int64_t clips) {
    if (states < 4) selective_step_kernel<T, 1, M, false><<<blocks, kThreads, 0, st>>>(a, state, clips);
    else if (states <= 16) selective_step_kernel<T, 1, M, true><<<blocks, kThreads, 0, st>>>(a, state, clips);
    else if (states <= 32) selective_step_kernel<T, 2, M, true><<<blocks, kThreads, 0, st>>>(a, state, clips);
    if constexpr (M == 1) {
        if (states > 64) selective_step_kernel<T, 8, M, true><<<blocks, kThreads, 0, st>>>(a, state, clips);
        else if (states > 32) selective_step_kernel<T, 4, M, true><<<blocks, kThreads, 0, st>>>(a, state, clips);
    }
}

}  // namespace

extern "C" {

size_t sedmi_selective_scan_workspace_bytes(int64_t n_clips, int64_t frames, int channels, int groups, int states) {
    if (!scan_shape_ok(n_clips, frames, channels, groups, states)) return 0;
    const int splits = scan_splits(n_clips, frames, channels, groups, states);
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
    const int waves = scan_waves(p->channels, p->groups, p->states);
    a.blocks_per_group = static_cast<int>(sedmi::ceil_div(a.per_group, 16 * waves));
    a.splits = scan_splits(p->n_clips, p->frames, p->channels, p->groups, p->states);
    a.run = scan_run(p->frames, a.splits);
    const size_t need = sedmi_selective_scan_workspace_bytes(p->n_clips, p->frames, p->channels, p->groups, p->states);
    if (need > 0 && (ws == nullptr || ws_bytes < need))
        return sedmi::set_error(SEDMI_ENOMEM, "selective_scan: workspace of %zu bytes, %zu needed", ws_bytes, need);
    a.end_state = static_cast<float *>(ws);
    a.end_step = a.end_state + static_cast<size_t>(p->n_clips) * (a.splits - 1) * p->channels * p->states;
    const int64_t per_clip = blocks_of(p->channels, p->groups, 16 * waves);
    SEDMI_REQUIRE(launch_ok(per_clip * a.splits, 64 * waves), "selective_scan: too many workgroups per clip");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const double items = static_cast<double>(p->n_clips) * p->frames * p->channels;
    const double es = p->dtype == SEDMI_DTYPE_F32 ? 4 : 2;
    return with_dtype(p->dtype, [&](auto t) -> int {
        using T = decltype(t);
        if (a.splits > 1) {                                      // few workgroups: one launch each
            {
                sedmi::ProfileScope scope("selective_scan_end_kernel", st, 5 * items * p->states, 2 * es * items);
                launch_scan<T, true>(p->states, waves, static_cast<unsigned>(p->n_clips * per_clip * (a.splits - 1)), st, a);
            }
            SEDMI_CHECK_LAUNCH();
        }
        {
            sedmi::ProfileScope scope("selective_scan_kernel", st, 7 * items * p->states, (p->z ? 4 : 3) * es * items);
            in_launches(p->n_clips, per_clip * a.splits, 64 * waves, [&](int64_t first, int64_t n) {
                launch_scan<T, false>(p->states, waves, static_cast<unsigned>(n * per_clip * a.splits), st, scan_args<T>(a, first));
            });
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
    ScanArgs a = scan_args(p);
    a.blocks_per_group = static_cast<int>(sedmi::ceil_div(a.per_group, kStepChannels));
    const int64_t per_clip = blocks_of(p->channels, p->groups, kStepChannels), blocks = p->n_clips * per_clip;
    SEDMI_REQUIRE(launch_ok(per_clip, kThreads), "selective_step: too many workgroups per stream");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const double items = static_cast<double>(p->n_clips) * p->channels;
    sedmi::ProfileScope scope("selective_step_kernel", st, 7 * items * p->states, 8 * items * p->states);
    // Four streams to a quad while that leaves two workgroups per compute unit and the states of four streams fit without
    // costing waves.  One against four streams (us): 256 x 2048 x 16 bf16 16.7 / 13.4, 256 x 4096 x 16 26.5 / 22.9,
    // 128 x 2048 x 64 24.2 / 26.3, 256 x 300 x 8 (1280 workgroups) 4.4 / 4.8.
    const bool four = blocks >= 2048 && p->states <= 32;
    return with_dtype(p->dtype, [&](auto t) -> int {
        using T = decltype(t);
        const int64_t each = four ? 4 : 1;                       // streams of a workgroup
        in_launches(sedmi::ceil_div(p->n_clips, each), per_clip, kThreads, [&](int64_t first, int64_t n) {
            const ScanArgs part = scan_args<T>(a, first * each);
            const int64_t streams = std::min(n * each, p->n_clips - first * each);
            if (four) launch_step<T, 4>(p->states, static_cast<unsigned>(n * per_clip), st, part, part.state_out, streams);
            else launch_step<T, 1>(p->states, static_cast<unsigned>(n * per_clip), st, part, part.state_out, streams);
        });
        SEDMI_CHECK_LAUNCH();
        return SEDMI_OK;
    });
}

}  // extern "C"
