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
constexpr int kMaxChunks = 256;         // of a clip's rows
constexpr int kUnroll = 4;               // rows of a thread in flight

struct NormArgs {
    const float *weight, *bias;          // [channels] or null
    const int64_t *lengths;              // [clips] or null
    int64_t frames, inner, rows;         // rows = frames * inner
    int channels, groups, per_group;     // per_group = channels / groups
    float eps;
    // two-launch form
    int groups_per_block, wider_blocks, column_blocks, chunks;  // the first wider_blocks have one group more
    int64_t rows_per_chunk;
    // one-launch form
    int vectors;                         // of a row of the group
    uint32_t per_row_inverse;            // floor(2^32 / vectors) + 1 (vectors > 1): i / vectors for i < 2^16
    float *partial;                      // [clips][chunks][groups][3] = count, mean, sum of squares about the mean
};

// Rows row, row + step, ... of `count` left from row on.
__device__ __forceinline__ int64_t rows_of(int64_t count, int step) { return count > 0 ? (count + step - 1) / step : 0; }

// Vectors side by side over `width` channels.  The last one of a width that is no multiple of V moves back over its
// neighbour's channels, `skip` of which it does not count; both write the same values there.  TINY (a width below V): one
// vector, loaded and stored by element.
template <typename T, bool TINY>
struct Column {
    static constexpr int V = kVec<T>;
    int at, skip, size;
    __device__ __forceinline__ Column(int j, int width) : at(TINY ? 0 : min(j * V, width - V)), skip(j * V - at), size(TINY ? width : V) {}
    __device__ __forceinline__ Pack<T, V> load(const T *p) const { return load_pack<T, V>(p + at, size); }
    __device__ __forceinline__ void store(T *p, const Pack<T, V> &v, bool stream) const {
        if (stream) stream_pack<T, V>(p + at, v, size);
        else store_pack<T, V>(p + at, v, size);
    }
    __device__ __forceinline__ bool counts(int e) const { return e >= skip && e < size; }
};

// --- two launches: statistics of row chunks, then their join and the rows themselves
//
// A thread keeps a running mean and a running sum of squares about it per channel (mean += d / n, m2 += d (x - mean)),
// which loses nothing where the mean is far from zero; one more operation per element than plain sums, in a kernel that
// waits for memory.  The rows are read twice, so its bytes are 3 / 2 of the one-launch form's: 128 x 250 x 8 x 128 bf16 with
// 32 groups 47 us (131 MB in and out), 64 x 250 x 1024 bf16 with one group 21, 1 x 251 x 387 f16 with gelu 11.
template <typename T, bool TINY>
__global__ __launch_bounds__(kThreads) void norm_stats_kernel(const T *x, NormArgs a) {
    constexpr int V = kVec<T>;
    // where vectors lie within a group: one entry per thread; else one per (row lane, channel)
    __shared__ float s_mean[kThreads * V], s_m2[kThreads * V], s_cnt[kThreads];
    const int tid = threadIdx.x;
    const int block = blockIdx.x % a.column_blocks;
    const int64_t rest = blockIdx.x / a.column_blocks;
    const int chunk = static_cast<int>(rest % a.chunks);
    const int64_t clip = rest / a.chunks;
    const int g0 = block * a.groups_per_block + min(block, a.wider_blocks);
    const int ng = a.groups_per_block + (block < a.wider_blocks);
    const int width = ng * a.per_group;                         // channels of this block
    const int nv = (width + V - 1) / V;
    const int64_t valid = clamp_length(a.lengths, clip, a.frames) * a.inner;
    const int64_t r0 = chunk * a.rows_per_chunk, r1 = min(valid, r0 + a.rows_per_chunk);
    const T *base = x + clip * a.rows * a.channels + static_cast<int64_t>(g0) * a.per_group;

    const int lanes = min(nv, kThreads);                        // threads side by side along a row
    const int rp = kThreads / lanes;
    const int row = tid / lanes, col = tid - row * lanes;
    const bool inside = ng == 1 || a.per_group % V == 0;        // always so where nv > kThreads (then ng == 1)
    float total_n = 0.0f, total_mean = 0.0f, total_m2 = 0.0f;
    for (int j = col; j < nv && row < rp; j += lanes) {
        const Column<T, TINY> c(j, width);
        float mean[V], m2[V], n = 0.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) mean[e] = m2[e] = 0.0f;
        const T *p = base + (r0 + row) * a.channels;
        const int64_t stride = static_cast<int64_t>(rp) * a.channels;
        auto add = [&](const Pack<T, V> &in) __attribute__((always_inline)) {
            n += 1.0f;
            const float inv = __builtin_amdgcn_rcpf(n);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float v = in.get(e), d = v - mean[e];
                mean[e] = fmaf(d, inv, mean[e]);
                m2[e] = fmaf(d, v - mean[e], m2[e]);
            }
        };
        int left = static_cast<int>(rows_of(r1 - r0 - row, rp));
        for (; left >= kUnroll; left -= kUnroll, p += kUnroll * stride) {
            Pack<T, V> in[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) in[u] = c.load(p + u * stride);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) add(in[u]);
        }
        if (left > 0) {                                          // the last rows together, the very last repeated
            Pack<T, V> in[kUnroll - 1];
#pragma unroll
            for (int u = 0; u < kUnroll - 1; ++u) in[u] = c.load(p + min(u, left - 1) * stride);
#pragma unroll
            for (int u = 0; u < kUnroll - 1; ++u)
                if (u < left) add(in[u]);
        }
        if (inside) {
            // the channels of the vector joined, all of count n, and those with what the thread has
            const float m = static_cast<float>(c.size - c.skip);
            float sum = 0.0f, q = 0.0f;
#pragma unroll
            for (int e = 0; e < V; ++e) sum += c.counts(e) ? mean[e] : 0.0f;
            const float middle = sum / m;
#pragma unroll
            for (int e = 0; e < V; ++e) q += c.counts(e) ? fmaf(n * (mean[e] - middle), mean[e] - middle, m2[e]) : 0.0f;
            const float all = total_n + n * m, d = middle - total_mean, w = all > 0.0f ? n * m / all : 0.0f;
            total_mean = fmaf(d, w, total_mean);
            total_m2 += fmaf(d * d, total_n * w, q);
            total_n = all;
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (c.counts(e)) {
                    s_mean[row * nv * V + c.at + e] = mean[e];
                    s_m2[row * nv * V + c.at + e] = m2[e];
                }
            if (j == 0) s_cnt[row] = n;
        }
    }
    // a group's entries: `entries` adjacent ones in each of `rows_in` rows of per_row
    int entries = a.per_group, per_row = nv * V, rows_in = rp;
    if (inside) {
        if (row < rp) s_mean[tid] = total_mean, s_m2[tid] = total_m2, s_cnt[tid] = total_n;
        entries = ng == 1 ? lanes : a.per_group / V, per_row = lanes;
    }
    __syncthreads();
    const int lane = tid & 63, wave = tid >> 6;
    const int first_r = lane / entries, first_e = lane - first_r * entries, step_r = 64 / entries, step_e = 64 - step_r * entries;
    auto walk = [&](int g, auto f) __attribute__((always_inline)) {
        for (int r = first_r, e = first_e; r < rows_in;) {
            const int at = r * per_row + g * entries + e;
            f(at, s_cnt[inside ? at : r]);
            r += step_r, e += step_e;
            if (e >= entries) e -= entries, ++r;
        }
    };
    for (int g = wave; g < ng; g += kThreads / 64) {
        float sum = 0.0f, cnt = 0.0f, m2 = 0.0f;
        walk(g, [&](int at, float n) { cnt += n, sum = fmaf(n, s_mean[at], sum); });
#pragma unroll
        for (int m = 32; m; m >>= 1) cnt += __shfl_xor(cnt, m), sum += __shfl_xor(sum, m);
        const float mean = cnt > 0.0f ? sum / cnt : 0.0f;
        walk(g, [&](int at, float n) { m2 += fmaf(n * (s_mean[at] - mean), s_mean[at] - mean, s_m2[at]); });
#pragma unroll
        for (int m = 32; m; m >>= 1) m2 += __shfl_xor(m2, m);
        if (lane == 0) {
            float *out = a.partial + ((clip * a.chunks + chunk) * a.groups + g0 + g) * 3;
            out[0] = cnt, out[1] = mean, out[2] = m2;
        }
    }
}

template <typename T, bool TINY, int ACT>
__global__ __launch_bounds__(kThreads) void norm_apply_kernel(const T *x, T *y, NormArgs a) {
    constexpr int V = kVec<T>;
    __shared__ float s_mean[kThreads * V], s_rstd[kThreads * V];
    const int tid = threadIdx.x;
    const int block = blockIdx.x % a.column_blocks;
    const int64_t rest = blockIdx.x / a.column_blocks;
    const int chunk = static_cast<int>(rest % a.chunks);
    const int64_t clip = rest / a.chunks;
    const int g0 = block * a.groups_per_block + min(block, a.wider_blocks);
    const int ng = a.groups_per_block + (block < a.wider_blocks);
    const int width = ng * a.per_group;
    const int nv = (width + V - 1) / V;
    const int64_t valid = clamp_length(a.lengths, clip, a.frames) * a.inner;
    const int64_t r0 = chunk * a.rows_per_chunk, r1 = min(a.rows, r0 + a.rows_per_chunk);
    const int64_t at0 = clip * a.rows * a.channels + static_cast<int64_t>(g0) * a.per_group;

    const int lanes = min(nv, kThreads);
    const int rp = kThreads / lanes;
    const int row = tid / lanes, col = tid - row * lanes;
    const int64_t stride = static_cast<int64_t>(rp) * a.channels, from = at0 + (r0 + row) * a.channels;
    const int rows = row < rp ? static_cast<int>(rows_of(r1 - r0 - row, rp)) : 0;
    const int good = row < rp ? static_cast<int>(rows_of(min(valid, r1) - r0 - row, rp)) : 0;
    Pack<T, V> in[kUnroll];
    auto fetch = [&](const Column<T, TINY> &c, int r) __attribute__((always_inline)) {       // rows past the last repeat it
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) in[u] = c.load(x + from + min(r + u, good - 1) * stride);
    };
    if (good > 0) fetch(Column<T, TINY>(col, width), 0);         // under way while the statistics are joined

    const int lane = tid & 63, wave = tid >> 6;
    for (int g = wave; g < ng; g += kThreads / 64) {
        constexpr int J = kMaxChunks / 64;                       // chunks of a lane
        float n[J], m[J], q[J], cnt = 0.0f, sum = 0.0f, m2 = 0.0f;
#pragma unroll
        for (int i = 0; i < J; ++i) {
            const bool on = lane + 64 * i < a.chunks;
            const float *p = a.partial + ((clip * a.chunks + min(lane + 64 * i, a.chunks - 1)) * a.groups + g0 + g) * 3;
            n[i] = p[0], m[i] = p[1], q[i] = p[2];
            if (!on) n[i] = m[i] = q[i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < J; ++i) cnt += n[i], sum = fmaf(n[i], m[i], sum);
#pragma unroll
        for (int k = 32; k; k >>= 1) cnt += __shfl_xor(cnt, k), sum += __shfl_xor(sum, k);
        const float mean = cnt > 0.0f ? sum / cnt : 0.0f;
#pragma unroll
        for (int i = 0; i < J; ++i) m2 += fmaf(n[i] * (m[i] - mean), m[i] - mean, q[i]);
#pragma unroll
        for (int k = 32; k; k >>= 1) m2 += __shfl_xor(m2, k);
        if (lane == 0) {
            s_mean[g] = mean;
            s_rstd[g] = 1.0f / sqrtf((cnt > 0.0f ? m2 / cnt : 0.0f) + a.eps);
        }
    }
    __syncthreads();

    for (int j = col; j < nv && rows > 0; j += lanes) {
        const Column<T, TINY> c(j, width);
        if (j != col && good > 0) fetch(c, 0);
        float mean[V], scale[V], shift[V];
        const auto w = a.weight ? load_pack<float, V>(a.weight + g0 * a.per_group + c.at, c.size) : Pack<float, V>::zero();
        const auto b = a.bias ? load_pack<float, V>(a.bias + g0 * a.per_group + c.at, c.size) : Pack<float, V>::zero();
        int g = c.at / a.per_group, next = (g + 1) * a.per_group - c.at;     // the element at which the next group begins
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (e == next && g + 1 < ng) ++g, next += a.per_group;
            mean[e] = s_mean[g];
            scale[e] = s_rstd[g] * (a.weight ? w.get(e) : 1.0f);
            shift[e] = b.get(e);
        }
        for (int r = 0; r < good; r += kUnroll) {
            Pack<T, V> out[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                float v[V];
#pragma unroll
                for (int e = 0; e < V; ++e)
                    v[e] = activate<ACT>(fmaf(in[u].get(e) - mean[e], scale[e], shift[e]));
                out[u] = Pack<T, V>::from(v);
            }
            if (r + kUnroll < good) fetch(c, r + kUnroll);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (r + u < good) c.store(y + from + (r + u) * stride, out[u], true);
        }
        for (int r = good; r < rows; ++r) c.store(y + from + r * stride, Pack<T, V>::zero(), true);
    }
}

// --- one launch: a clip's group of at least V channels fits into the registers of a workgroup
//
// x is read once and held as it is in memory; mean, then the squares about it, then the output.  Workgroups of the groups
// of one clip follow each other on one die (blocks are dealt to the 8 dies in turn), so lines that two groups share are
// fetched into one L2: by the counters every byte is read once.  Groups of 32-byte rows (128 x 250 x 16 x 64 f32, 8 groups)
// also write every byte once, 75 us, 3.5 TB/s.  Groups of 64-byte rows (64 x 250 x 1024 bf16, 32 groups) take 18 us,
// 3.6 TB/s, and with half of the frames behind the lengths 15.5; they write a quarter more than the output has (40.8 of
// 32.0 thousand KiB), with stores past L2 of half a 128-byte line each.  A workgroup reads, sums and writes in turn; twice
// the workgroups per compute unit (90 us for the first shape) and a loop that loads the next group early into registers
// (84 us) need more registers than there are and lose.
template <typename T, int N, int ACT>
__global__ __launch_bounds__(1024) void norm_slab_kernel(const T *x, T *y, NormArgs a) {
    constexpr int V = kVec<T>;
    __shared__ float s_sum[2][16];
    const int tid = threadIdx.x, threads = blockDim.x;
    const unsigned per_die = gridDim.x / 8, dealt = per_die * 8;
    const unsigned block = blockIdx.x < dealt ? (blockIdx.x % 8) * per_die + blockIdx.x / 8 : blockIdx.x;
    const int64_t clip = block / a.groups;
    const int c0 = (block - static_cast<unsigned>(clip) * a.groups) * a.per_group;
    const int rows = static_cast<int>(a.rows);
    const int good = static_cast<int>(clamp_length(a.lengths, clip, a.frames) * a.inner);       // valid rows
    const T *px = x + clip * a.rows * a.channels + c0;
    T *py = y + clip * a.rows * a.channels + c0;

    auto row_of = [&](int k) __attribute__((always_inline)) {
        const unsigned i = tid + k * threads;
        return static_cast<int>(a.vectors == 1 ? i : __umulhi(i, a.per_row_inverse));
    };
    auto column_of = [&](int k, int row) __attribute__((always_inline)) {
        return Column<T, false>(tid + k * threads - row * a.vectors, a.per_group);
    };
    Pack<T, V> in[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int row = row_of(k);                               // rows behind the last valid one repeat it, uncounted
        in[k] = Pack<T, V>::zero();
        if (good > 0) in[k] = column_of(k, row).load(px + static_cast<int64_t>(min(row, good - 1)) * a.channels);
    }
    auto skip_of = [&](int k) __attribute__((always_inline)) {
        const int row = row_of(k);
        return row < good ? column_of(k, row).skip : V;
    };
    // unpacked anew in each phase: kept as float32 between them, the rows would need twice the registers
    auto repack = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int i = 0; i < V / Pack<T, V>::kPer; ++i) asm volatile("" : "+v"(in[k].w[i]));
    };
    auto total = [&](float v, float *s) __attribute__((always_inline)) {
#pragma unroll
        for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
        if ((tid & 63) == 0) s[tid >> 6] = v;
        __syncthreads();
        float t = 0.0f;
        for (int i = 0; i < threads / 64; ++i) t += s[i];
        return t;
    };
    float sum = 0.0f, squares = 0.0f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int skip = skip_of(k);
#pragma unroll
        for (int e = 0; e < V; ++e) sum += e >= skip ? in[k].get(e) : 0.0f;
    }
    const float items = fmaxf(static_cast<float>(good) * static_cast<float>(a.per_group), 1.0f);
    const float mean = total(sum, s_sum[0]) / items;
    repack();
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int skip = skip_of(k);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float d = in[k].get(e) - mean;
            squares += e >= skip ? d * d : 0.0f;
        }
    }
    const float rstd = 1.0f / sqrtf(total(squares, s_sum[1]) / items + a.eps);
    repack();
    const bool one_column = threads % a.vectors == 0;            // all vectors of a thread lie in the same channels
    Pack<float, V> w = Pack<float, V>::zero(), b = w;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int row = row_of(k);
        const auto c = column_of(k, row);
        if (k == 0 || !one_column) {
            if (a.weight) w = load_pack<float, V>(a.weight + c0 + c.at, V);
            if (a.bias) b = load_pack<float, V>(a.bias + c0 + c.at, V);
        }
        if (row >= rows) continue;
        float v[V];
#pragma unroll
        for (int e = 0; e < V; ++e)
            v[e] = activate<ACT>(fmaf((in[k].get(e) - mean) * rstd, a.weight ? w.get(e) : 1.0f, b.get(e)));
        c.store(py + static_cast<int64_t>(row) * a.channels, row < good ? Pack<T, V>::from(v) : Pack<T, V>::zero(),
                a.per_group * sizeof(T) >= 64);
    }
}

// Row chunks and column blocks of the two-launch form.
struct NormPlan {
    int groups_per_block, wider_blocks, column_blocks, chunks;
    int64_t rows_per_chunk;
    bool tiny;                           // fewer channels than a vector
};

NormPlan norm_plan(int64_t clips, int64_t rows, int channels, int groups, int vec) {
    NormPlan p;
    const int per_group = channels / groups;
    // Blocks of at most kThreads vectors, the groups dealt out evenly: more than half of the widest possible block goes to
    // each of several, so none is narrower than a vector.
    const int fit = std::max(1, std::min(groups, kThreads * vec / per_group));
    p.column_blocks = static_cast<int>(sedmi::ceil_div(groups, fit));
    p.groups_per_block = groups / p.column_blocks;
    p.wider_blocks = groups % p.column_blocks;
    p.tiny = channels < vec;
    const int widest = p.groups_per_block + (p.wider_blocks > 0);
    const int nv = std::min<int64_t>(kThreads, sedmi::ceil_div(static_cast<int64_t>(widest) * per_group, vec));
    const int64_t rp = kThreads / nv;
    // Every workgroup joins statistics, so few: two per compute unit (128 x 250 x 8 x 128 with 32 groups, bf16: 512 53 us,
    // 1024 57, 2048 74), and no less than kUnroll rows for each of its threads.
    const int64_t want = sedmi::ceil_div(512, std::max<int64_t>(1, clips * p.column_blocks));
    const int64_t most = std::max<int64_t>(1, rows / (rp * kUnroll));
    p.chunks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, most, kMaxChunks})));
    p.rows_per_chunk = sedmi::ceil_div(std::max<int64_t>(rows, 1), p.chunks);
    return p;
}

int dtype_vec(int dtype) { return dtype == SEDMI_DTYPE_F32 ? 4 : 8; }

// Whether a clip's group is normalised by one workgroup in one launch: up to 64 KiB of it, and up to 128 KiB where there
// are workgroups for every compute unit (a single unit takes 5 us for the second 64 KiB).  Measured, one launch against two
// (us): 64 x 32 groups of 16 kB bf16 19.2 / 59, 1 x 64 KiB 8.9 / 9.2, 128 x 64 KiB 10.4 / 12.2, 64 x 128 KiB 16.0 / 12.3,
// 256 x 128 KiB 21.2 / 22.4, 1024 x 128 KiB f32 81 / 86, 64 x 256 KiB 28 / 16.
bool use_slab(int64_t clips, int64_t rows, int channels, int groups, int vec) {
    const int per_group = channels / groups;
    const int64_t vectors = rows * sedmi::ceil_div(per_group, vec);
    return per_group >= vec && launch_ok(groups, 1024) && (vectors <= 4096 || (vectors <= 8192 && clips * groups >= 256));
}

template <typename T>
void launch_slab(const T *x, T *y, NormArgs a, int64_t clips, int activation, hipStream_t st) {
    a.vectors = static_cast<int>(sedmi::ceil_div(a.per_group, kVec<T>));
    a.per_row_inverse = a.vectors > 1 ? static_cast<uint32_t>((uint64_t{1} << 32) / a.vectors + 1) : 0;
    const int64_t vectors = a.rows * a.vectors;
    const int threads = vectors <= 512 ? 256 : vectors <= 1024 ? 512 : 1024;       // up to 2 vectors each, then up to 8
    const int64_t each = sedmi::ceil_div(vectors, threads), clip = a.rows * a.channels;
    in_launches(clips, a.groups, threads, [&](int64_t first, int64_t n) {
        const unsigned blocks = static_cast<unsigned>(n * a.groups);
        with_activation(activation, [&](auto act) {
            constexpr int kAct = decltype(act)::value;
            const T *px = x + first * clip;
            T *py = y + first * clip;
            if (each <= 1) norm_slab_kernel<T, 1, kAct><<<blocks, threads, 0, st>>>(px, py, a);
            else if (each <= 2) norm_slab_kernel<T, 2, kAct><<<blocks, threads, 0, st>>>(px, py, a);
            else if (each <= 4) norm_slab_kernel<T, 4, kAct><<<blocks, threads, 0, st>>>(px, py, a);
            else norm_slab_kernel<T, 8, kAct><<<blocks, threads, 0, st>>>(px, py, a);
        });
        if (a.lengths) a.lengths += n;
    });
}

bool norm_shape_ok(int64_t clips, int64_t frames, int64_t inner, int channels, int groups, int dtype) {
    return frames >= 0 && inner > 0 && frames <= (int64_t{1} << 38) / inner &&
           sequence_shape_ok(clips, frames * inner, channels) && groups > 0 && channels % groups == 0 && dtype_ok(dtype);
}

}  // namespace

extern "C" {

size_t sedmi_group_norm_workspace_bytes(int64_t n_clips, int64_t frames, int64_t inner, int channels, int groups,
                                        int dtype) {
    if (!norm_shape_ok(n_clips, frames, inner, channels, groups, dtype)) return 0;
    if (use_slab(n_clips, frames * inner, channels, groups, dtype_vec(dtype))) return 0;
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
    a.eps = eps;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const double items = static_cast<double>(n_clips) * a.rows * channels;
    const double es = dtype == SEDMI_DTYPE_F32 ? 4 : 2;
    if (use_slab(n_clips, a.rows, channels, groups, dtype_vec(dtype))) {
        sedmi::ProfileScope scope("norm_slab_kernel", st, 8 * items, 2 * es * items);
        with_dtype(dtype, [&](auto t) -> int {
            launch_slab(static_cast<const decltype(t) *>(x), static_cast<decltype(t) *>(y), a, n_clips, activation, st);
            return SEDMI_OK;
        });
        SEDMI_CHECK_LAUNCH();
        return SEDMI_OK;
    }
    const NormPlan p = norm_plan(n_clips, a.rows, channels, groups, dtype_vec(dtype));
    a.groups_per_block = p.groups_per_block, a.wider_blocks = p.wider_blocks, a.column_blocks = p.column_blocks;
    a.chunks = p.chunks, a.rows_per_chunk = p.rows_per_chunk;
    const int64_t per_clip = static_cast<int64_t>(p.chunks) * p.column_blocks;       // at most 2^8 * 2^14
    const size_t need = static_cast<size_t>(n_clips) * p.chunks * groups * 3 * sizeof(float);
    if (ws == nullptr || ws_bytes < need)
        return sedmi::set_error(SEDMI_ENOMEM, "group_norm: workspace of %zu bytes, %zu needed", ws_bytes, need);
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        in_launches(n_clips, per_clip, kThreads, [&](int64_t first, int64_t n) {
            const unsigned grid = static_cast<unsigned>(n * per_clip);
            const T *px = static_cast<const T *>(x) + first * a.rows * channels;
            T *py = static_cast<T *>(y) + first * a.rows * channels;
            const double share = static_cast<double>(n) / n_clips;
            a.lengths = lengths ? lengths + first : nullptr;
            a.partial = static_cast<float *>(ws) + first * p.chunks * groups * 3;
            {
                sedmi::ProfileScope scope("norm_stats_kernel", st, share * 4 * items, share * es * items);
                if (p.tiny) norm_stats_kernel<T, true><<<grid, kThreads, 0, st>>>(px, a);
                else norm_stats_kernel<T, false><<<grid, kThreads, 0, st>>>(px, a);
            }
            sedmi::ProfileScope scope("norm_apply_kernel", st, share * 4 * items, share * 2 * es * items);
            with_activation(activation, [&](auto act) {
                constexpr int kAct = decltype(act)::value;
                if (p.tiny) norm_apply_kernel<T, true, kAct><<<grid, kThreads, 0, st>>>(px, py, a);
                else norm_apply_kernel<T, false, kAct><<<grid, kThreads, 0, st>>>(px, py, a);
            });
        });
        SEDMI_CHECK_LAUNCH();
        return SEDMI_OK;
    });
}

}  // extern "C"
