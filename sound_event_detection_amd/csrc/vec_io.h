// Element types and 16-byte row access of the channels-last sequence operators (norm.hip, conv1d.hip, scan.hip).  Meant to
// be included INSIDE an anonymous namespace of the including translation unit.
#pragma once

// Longest vector a lane moves in one instruction: 16 bytes.
template <typename T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));

// Two 16-bit elements of a word, or one float32 word.
template <typename T>
__device__ __forceinline__ float element(uint32_t w, int i);
template <>
__device__ __forceinline__ float element<float>(uint32_t w, int) { return __builtin_bit_cast(float, w); }
template <>
__device__ __forceinline__ float element<__bf16>(uint32_t w, int i) {
    return __builtin_bit_cast(float, i ? w & 0xffff0000u : w << 16);
}
template <>
__device__ __forceinline__ float element<_Float16>(uint32_t w, int i) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(i ? w >> 16 : w)));
}

// V elements as the 32-bit words they are in memory: unpacked where they are used, so that a row in flight costs no more
// registers than it has bytes.  A row of an odd number of elements, or of a slice of a projection, starts at any multiple
// of the element size.  The hardware takes unaligned 16-byte global accesses (gfx950 under ROCm runs with unaligned
// access on), so one code path serves every alignment: the type only promises the alignment of an element.
template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
    static constexpr int kPer = 4 / static_cast<int>(sizeof(T));         // elements per word
    uint32_t w[V / kPer];

    __device__ __forceinline__ float get(int e) const { return element<T>(w[e / kPer], e % kPer); }
    __device__ __forceinline__ static Pack zero() {
        Pack r;
#pragma unroll
        for (int i = 0; i < V / kPer; ++i) r.w[i] = 0;
        return r;
    }
    // word i from its elements, rounded to nearest even
    __device__ __forceinline__ void set_word(int i, const float *v) {
        if constexpr (kPer == 1) {
            w[i] = __builtin_bit_cast(uint32_t, v[0]);
        } else {
            using F2 = __attribute__((ext_vector_type(2))) float;
            using T2 = __attribute__((ext_vector_type(2))) T;
            w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((F2{v[0], v[1]}), T2));
        }
    }
    __device__ __forceinline__ static Pack from(const float *v) {
        Pack r;
#pragma unroll
        for (int i = 0; i < V / kPer; ++i) r.set_word(i, v + i * kPer);
        return r;
    }
};

template <typename T>
using Bits = std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t>;

// The first n of V elements at p, 1 <= n: one load, or for the last elements of a row single loads of which those past
// the end repeat the last element (no branch each, so all are in flight together; what they hold is never stored).
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T *p, int n) {
    Pack<T, V> r;
    if (n >= V) {
        r = *reinterpret_cast<const Pack<T, V> *>(p);
    } else {
        const Bits<T> *b = reinterpret_cast<const Bits<T> *>(p);
#pragma unroll
        for (int i = 0; i < V / r.kPer; ++i) {
            r.w[i] = b[min(i * r.kPer, n - 1)];
            if constexpr (sizeof(T) == 2) r.w[i] |= static_cast<uint32_t>(b[min(2 * i + 1, n - 1)]) << 16;
        }
    }
    return r;
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, V> &r, int n) {
    if (n >= V) {
        *reinterpret_cast<Pack<T, V> *>(p) = r;
    } else {
        Bits<T> *b = reinterpret_cast<Bits<T> *>(p);
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < n) b[e] = static_cast<Bits<T>>(r.w[e / r.kPer] >> (sizeof(T) == 2 ? 16 * (e % 2) : 0));
    }
}

// The same for an output that the kernel does not touch again: a store that does not stay in L2 leaves it to the inputs
// (us: convolution of 128 x 250 x 2048 bf16 61 -> 58, 16 x 1000 x 2047 33 -> 28; norm of 128 x 250 x 8 x 128 53 -> 47).  For
// rows that are written in one go: with pieces of 32 bytes it takes longer (norm of 128 x 250 x 16 x 64 f32, 8 groups: 81 ->
// 140).  The same on loads loses everywhere (norm of 64 x 250 x 1024, 32 groups: 18 -> 27), as neighbours share lines.
template <typename T, int V>
__device__ __forceinline__ void stream_pack(T *p, const Pack<T, V> &r, int n) {
    constexpr int W = V / Pack<T, V>::kPer;
    if (n >= V) {
        using Words = uint32_t __attribute__((ext_vector_type(W), aligned(sizeof(T))));
        Words w;
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = r.w[i];
        __builtin_nontemporal_store(w, reinterpret_cast<Words *>(p));
    } else {
        store_pack<T, V>(p, r, n);
    }
}

// 0 from x = -87.4 down, where the reciprocal is below 2^-126 (the value is above -1.3e-36 there).
__device__ __forceinline__ float silu(float x) { return x * __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

// x Phi(x) = max(x, 0) - |x| erfc(z) / 2 with z = |x| / sqrt 2, which cancels nowhere.  erfc(z) = exp(-z^2) t Q(t),
// t = 1 / (1 + z / 2), Q the polynomial of degree 8 nearest to exp(z^2) erfc(z) / t for z <= 12 (4.4e-8 of it; 3.1e-7 as
// evaluated).  No branch, where a library erf has one per range (norm of 1 x 251 x 387 f16: 14.9 -> 11.2 us).
__device__ __forceinline__ float gelu(float x) {
    const float z = fabsf(x) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(fmaf(0.5f, z, 1.0f));
    float q = fmaf(-0.059363074600696564f, t, 0.2860105633735657f);
    q = fmaf(q, t, -0.4901731610298157f);
    q = fmaf(q, t, 0.28146857023239136f);
    q = fmaf(q, t, -0.028967853635549545f);
    q = fmaf(q, t, 0.20367690920829773f);
    q = fmaf(q, t, 0.24285396933555603f);
    q = fmaf(q, t, 0.28240954875946045f);
    q = fmaf(q, t, 0.28208446502685547f);
    const float rest = 0.5f * fabsf(x) * (t * q * __builtin_amdgcn_exp2f(-1.44269504088896341f * z * z));
    return fmaxf(x, 0.0f) - (x > 14.0f ? 0.0f : rest);           // erfc(14 / sqrt 2) is below 2^-126; infinity stays
}

// ACT: a SEDMI_ACT_* code (sedmi.h).
template <int ACT>
__device__ __forceinline__ float activate(float x) {
    if constexpr (ACT == SEDMI_ACT_RELU) return x < 0.0f ? 0.0f : x;      // NaN stays NaN
    else if constexpr (ACT == SEDMI_ACT_SILU) return silu(x);
    else if constexpr (ACT == SEDMI_ACT_GELU) return gelu(x);
    else return x;
}

__device__ __forceinline__ int64_t clamp_length(const int64_t *lengths, int64_t i, int64_t most) {
    if (lengths == nullptr) return most;
    const int64_t n = lengths[i];
    return n < 0 ? 0 : (n > most ? most : n);
}

inline bool dtype_ok(int dtype) {
    return dtype == SEDMI_DTYPE_F32 || dtype == SEDMI_DTYPE_F16 || dtype == SEDMI_DTYPE_BF16;
}

// Limits that keep every offset, in bytes too, below 2^63.
inline bool sequence_shape_ok(int64_t clips, int64_t frames, int64_t channels) {
    return clips >= 0 && clips <= (int64_t{1} << 22) && channels > 0 && channels <= (1 << 24) && frames >= 0 &&
           frames <= (int64_t{1} << 38) / channels;
}

inline bool overlap(const void *p, const void *q, size_t bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(p), y = reinterpret_cast<uintptr_t>(q);
    return p != nullptr && q != nullptr && x < y + bytes && y < x + bytes;
}

// A launch has fewer than 2^32 lanes: HIP counts them in 32 bits.
constexpr int64_t kMaxLanes = (int64_t{1} << 32) - 1;

inline bool launch_ok(int64_t blocks, int threads) { return blocks <= kMaxLanes / threads; }

// Calls f(first clip, clips) for as many clips at a time as a launch of that many workgroups each can hold; a single clip's
// have to be launch_ok.
template <typename F>
void in_launches(int64_t clips, int64_t blocks_per_clip, int threads, F f) {
    const int64_t most = kMaxLanes / threads / blocks_per_clip;
    for (int64_t first = 0; first < clips; first += most) f(first, std::min(most, clips - first));
}

// Dispatches f(T{}) on a SEDMI_DTYPE_* code.
template <typename F>
int with_dtype(int dtype, F f) {
    if (dtype == SEDMI_DTYPE_F32) return f(float{});
    if (dtype == SEDMI_DTYPE_F16) return f(static_cast<_Float16>(0.0f));
    return f(static_cast<__bf16>(0.0f));
}

// Calls f with the activation as a constant: looked up per element, its branches keep elements from overlapping.
template <typename F>
void with_activation(int act, F f) {
    if (act == SEDMI_ACT_RELU) f(std::integral_constant<int, SEDMI_ACT_RELU>{});
    else if (act == SEDMI_ACT_SILU) f(std::integral_constant<int, SEDMI_ACT_SILU>{});
    else if (act == SEDMI_ACT_GELU) f(std::integral_constant<int, SEDMI_ACT_GELU>{});
    else f(std::integral_constant<int, SEDMI_ACT_NONE>{});
}
