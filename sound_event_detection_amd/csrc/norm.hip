// Group normalisation with an activation on channels-last activations [clips, frames, inner, channels]:
//
//     y = act((x - m) / sqrt(v + eps) * weight[c] + bias[c])
//
// with m and v the mean and the biased variance of a clip's group of channels / groups channels over its valid rows
// (a row = one (frame, inner) position; frames at and behind lengths[clip] are neither read nor counted, their
// outputs are zero).
#include "common.h"

#include <algorithm>
#include <type_traits>

namespace {
#include "vec_io.h"

constexpr int kThreads = 256;

struct NormArgs {
    const float *weight, *bias;          // [channels] or null
    const int64_t *lengths;              // [clips] or null
    int64_t frames, inner, rows;         // rows = frames * inner
    int channels, groups, per_group;     // per_group = channels / groups
    float eps;
    int act;
    // two-launch form
    int groups_per_block, column_blocks, chunks;
    int64_t rows_per_chunk;
    float *partial;                      // [clips][chunks][groups][3] = count, mean, sum of squares about the mean
};

template <typename T>
__global__ __launch_bounds__(kThreads) void norm_stats_kernel(const T *x, NormArgs a) {
    constexpr int V = kVec<T>;
    __shared__ float s_mean[kThreads * V], s_m2[kThreads * V], s_cnt[kThreads];
    const int tid = threadIdx.x;
    const int block = blockIdx.x % a.column_blocks;
    const int64_t rest = blockIdx.x / a.column_blocks;
    const int chunk = static_cast<int>(rest % a.chunks);
    const int64_t clip = rest / a.chunks;
    const int g0 = block * a.groups_per_block;
    const int ng = min(a.groups_per_block, a.groups - g0);
    const int width = ng * a.per_group;                         // channels of this block
    const int nv = (width + V - 1) / V;
    const int64_t valid = clamp_length(a.lengths, clip, a.frames) * a.inner;
    const int64_t r0 = chunk * a.rows_per_chunk, r1 = min(valid, r0 + a.rows_per_chunk);
    const T *base = x + clip * a.rows * a.channels + static_cast<int64_t>(g0) * a.per_group;

    const int lanes = min(nv, kThreads);                        // threads side by side along a row
    const int rp = kThreads / lanes;
    const int row = tid / lanes, col = tid - row * lanes;
    float total_n = 0.0f, total_mean = 0.0f, total_m2 = 0.0f;   // one group wider than the workgroup: merged over its columns
    for (int j = col; j < nv; j += lanes) {
        const int ne = min(V, width - j * V);
        float mean[V], m2[V], n = 0.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) mean[e] = m2[e] = 0.0f;
        if (row < rp) {
            for (int64_t r = r0 + row; r < r1; r += rp) {
                const auto p = load_pack<T, V>(base + r * a.channels + j * V, ne);
                n += 1.0f;
                const float inv = __builtin_amdgcn_rcpf(n);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float v = p.get(e), d = v - mean[e];
                    mean[e] = fmaf(d, inv, mean[e]);
                    m2[e] = fmaf(d, v - mean[e], m2[e]);
                }
            }
        }
        if (nv > kThreads) {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (e < ne && n > 0.0f) {
                    const float sum = total_n + n, d = mean[e] - total_mean, w = n / sum;
                    total_mean = fmaf(d, w, total_mean);
                    total_m2 += m2[e] + d * d * total_n * w;
                    total_n = sum;
                }
        } else if (row < rp) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                s_mean[(row * nv + j) * V + e] = mean[e];
                s_m2[(row * nv + j) * V + e] = m2[e];
            }
            s_cnt[row * nv + j] = n;
        }
    }
    int entries = a.per_group, per_row = nv * V, rows_in = rp;  // entries of one group in a row of the tables
    if (nv > kThreads) {
        s_mean[tid] = total_mean, s_m2[tid] = total_m2, s_cnt[tid] = total_n;
        entries = kThreads, per_row = kThreads, rows_in = 1;
    }
    __syncthreads();
    const int lane = tid & 63, wave = tid >> 6;
    for (int g = wave; g < ng; g += kThreads / 64) {
        float sum = 0.0f, cnt = 0.0f;
        for (int i = lane; i < entries * rows_in; i += 64) {
            const int r = i / entries, at = r * per_row + g * entries + (i - r * entries);
            const float n = nv > kThreads ? s_cnt[at] : s_cnt[at / V];
            cnt += n;
            sum = fmaf(n, s_mean[at], sum);
        }
#pragma unroll
        for (int m = 32; m; m >>= 1) cnt += __shfl_xor(cnt, m), sum += __shfl_xor(sum, m);
        const float mean = cnt > 0.0f ? sum / cnt : 0.0f;
        float m2 = 0.0f;
        for (int i = lane; i < entries * rows_in; i += 64) {
            const int r = i / entries, at = r * per_row + g * entries + (i - r * entries);
            const float n = nv > kThreads ? s_cnt[at] : s_cnt[at / V], d = s_mean[at] - mean;
            m2 += s_m2[at] + n * d * d;
        }
#pragma unroll
        for (int m = 32; m; m >>= 1) m2 += __shfl_xor(m2, m);
        if (lane == 0) {
            float *out = a.partial + ((clip * a.chunks + chunk) * a.groups + g0 + g) * 3;
            out[0] = cnt, out[1] = mean, out[2] = m2;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void norm_apply_kernel(const T *x, T *y, NormArgs a) {
    constexpr int V = kVec<T>;
    __shared__ float s_mean[kThreads * V], s_rstd[kThreads * V];
    const int tid = threadIdx.x;
    const int block = blockIdx.x % a.column_blocks;
    const int64_t rest = blockIdx.x / a.column_blocks;
    const int chunk = static_cast<int>(rest % a.chunks);
    const int64_t clip = rest / a.chunks;
    const int g0 = block * a.groups_per_block;
    const int ng = min(a.groups_per_block, a.groups - g0);
    const int width = ng * a.per_group;
    const int nv = (width + V - 1) / V;
    const int64_t valid = clamp_length(a.lengths, clip, a.frames) * a.inner;
    const int64_t r0 = chunk * a.rows_per_chunk, r1 = min(a.rows, r0 + a.rows_per_chunk);
    const int64_t at0 = clip * a.rows * a.channels + static_cast<int64_t>(g0) * a.per_group;

    const int lane = tid & 63, wave = tid >> 6;
    for (int g = wave; g < ng; g += kThreads / 64) {             // chunks <= 64: one lane each
        float n = 0.0f, m = 0.0f, q = 0.0f;
        if (lane < a.chunks) {
            const float *p = a.partial + ((clip * a.chunks + lane) * a.groups + g0 + g) * 3;
            n = p[0], m = p[1], q = p[2];
        }
        float cnt = n, sum = n * m;
#pragma unroll
        for (int k = 32; k; k >>= 1) cnt += __shfl_xor(cnt, k), sum += __shfl_xor(sum, k);
        const float mean = cnt > 0.0f ? sum / cnt : 0.0f;
        float m2 = q + n * (m - mean) * (m - mean);
#pragma unroll
        for (int k = 32; k; k >>= 1) m2 += __shfl_xor(m2, k);
        if (lane == 0) {
            s_mean[g] = mean;
            s_rstd[g] = 1.0f / sqrtf((cnt > 0.0f ? m2 / cnt : 0.0f) + a.eps);
        }
    }
    __syncthreads();

    const int lanes = min(nv, kThreads);
    const int rp = kThreads / lanes;
    const int row = tid / lanes, col = tid - row * lanes;
    if (row >= rp) return;
    for (int j = col; j < nv; j += lanes) {
        const int ne = min(V, width - j * V);
        float mean[V], scale[V], shift[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int c = min(j * V + e, width - 1), g = c / a.per_group, ch = g0 * a.per_group + c;
            mean[e] = s_mean[g];
            scale[e] = s_rstd[g] * (a.weight ? a.weight[ch] : 1.0f);
            shift[e] = a.bias ? a.bias[ch] : 0.0f;
        }
        for (int64_t r = r0 + row; r < r1; r += rp) {
            const int64_t at = at0 + r * a.channels + j * V;
            Pack<T, V> out = Pack<T, V>::zero();
            if (r < valid) {
                const auto p = load_pack<T, V>(x + at, ne);
                float v[V];
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = activate(fmaf(p.get(e) - mean[e], scale[e], shift[e]), a.act);
                out = Pack<T, V>::from(v);
            }
            store_pack<T, V>(y + at, out, ne);
        }
    }
}

// Row chunks and column blocks of the two-launch form.
struct NormPlan {
    int groups_per_block, column_blocks, chunks;
    int64_t rows_per_chunk;
};

NormPlan norm_plan(int64_t clips, int64_t rows, int channels, int groups, int vec) {
    NormPlan p;
    const int per_group = channels / groups;
    p.groups_per_block = std::max(1, std::min(groups, kThreads * vec / per_group));
    p.column_blocks = static_cast<int>(sedmi::ceil_div(groups, p.groups_per_block));
    const int nv = std::min<int64_t>(kThreads, sedmi::ceil_div(static_cast<int64_t>(p.groups_per_block) * per_group, vec));
    const int64_t rp = kThreads / nv;
    const int64_t want = sedmi::ceil_div(2048, std::max<int64_t>(1, clips * p.column_blocks));
    const int64_t most = std::max<int64_t>(1, rows / (rp * 8));
    p.chunks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, most, 64})));
    p.rows_per_chunk = sedmi::ceil_div(std::max<int64_t>(rows, 1), p.chunks);
    return p;
}

int dtype_vec(int dtype) { return dtype == SEDMI_DTYPE_F32 ? 4 : 8; }

bool norm_shape_ok(int64_t clips, int64_t frames, int64_t inner, int channels, int groups, int dtype) {
    return clips >= 0 && frames >= 0 && inner > 0 && channels > 0 && groups > 0 && channels % groups == 0 &&
           (dtype == SEDMI_DTYPE_F32 || dtype == SEDMI_DTYPE_F16 || dtype == SEDMI_DTYPE_BF16) &&
           frames <= (int64_t{1} << 40) / inner && frames * inner <= (int64_t{1} << 40) / channels &&
           clips <= (int64_t{1} << 24);
}

}  // namespace

extern "C" {

size_t sedmi_group_norm_workspace_bytes(int64_t n_clips, int64_t frames, int64_t inner, int channels, int groups,
                                        int dtype) {
    if (!norm_shape_ok(n_clips, frames, inner, channels, groups, dtype)) return 0;
    const NormPlan p = norm_plan(n_clips, frames * inner, channels, groups, dtype_vec(dtype));
    return static_cast<size_t>(n_clips) * p.chunks * groups * 3 * sizeof(float);
}

int sedmi_group_norm(const void *x, const float *weight, const float *bias, const int64_t *lengths, void *y,
                     int64_t n_clips, int64_t frames, int64_t inner, int channels, int groups, float eps,
                     int activation, int dtype, void *ws, size_t ws_bytes, void *stream) {
    SEDMI_REQUIRE(channels > 0 && groups > 0 && channels % groups == 0,
                  "group_norm: channels (%d) must be a positive multiple of groups (%d)", channels, groups);
    SEDMI_REQUIRE(norm_shape_ok(n_clips, frames, inner, channels, groups, dtype),
                  "group_norm: bad shape or dtype (clips %lld, frames %lld, inner %lld, dtype %d)",
                  static_cast<long long>(n_clips), static_cast<long long>(frames), static_cast<long long>(inner), dtype);
    SEDMI_REQUIRE(activation >= SEDMI_ACT_NONE && activation <= SEDMI_ACT_GELU, "group_norm: unknown activation %d", activation);
    SEDMI_REQUIRE(eps >= 0.0f, "group_norm: eps must not be negative");
    if (n_clips == 0 || frames == 0) return SEDMI_OK;
    SEDMI_REQUIRE(x != nullptr && y != nullptr, "group_norm: null x or y");
    NormArgs a{};
    a.weight = weight, a.bias = bias, a.lengths = lengths;
    a.frames = frames, a.inner = inner, a.rows = frames * inner;
    a.channels = channels, a.groups = groups, a.per_group = channels / groups;
    a.eps = eps, a.act = activation;
    const NormPlan p = norm_plan(n_clips, a.rows, channels, groups, dtype_vec(dtype));
    a.groups_per_block = p.groups_per_block, a.column_blocks = p.column_blocks;
    a.chunks = p.chunks, a.rows_per_chunk = p.rows_per_chunk;
    const int64_t blocks = n_clips * p.chunks * p.column_blocks;
    SEDMI_REQUIRE(blocks < (int64_t{1} << 31), "group_norm: too many workgroups (%lld)", static_cast<long long>(blocks));
    const size_t need = static_cast<size_t>(n_clips) * p.chunks * groups * 3 * sizeof(float);
    if (ws == nullptr || ws_bytes < need)
        return sedmi::set_error(SEDMI_ENOMEM, "group_norm: workspace of %zu bytes, %zu needed", ws_bytes, need);
    a.partial = static_cast<float *>(ws);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const double items = static_cast<double>(n_clips) * a.rows * channels;
    const double es = dtype == SEDMI_DTYPE_F32 ? 4 : 2;
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        {
            sedmi::ProfileScope scope("norm_stats_kernel", st, 4 * items, es * items);
            norm_stats_kernel<T><<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(static_cast<const T *>(x), a);
        }
        SEDMI_CHECK_LAUNCH();
        {
            sedmi::ProfileScope scope("norm_apply_kernel", st, 4 * items, 2 * es * items);
            norm_apply_kernel<T><<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(static_cast<const T *>(x),
                                                                                      static_cast<T *>(y), a);
        }
        SEDMI_CHECK_LAUNCH();
        return SEDMI_OK;
    });
}

}  // extern "C"
