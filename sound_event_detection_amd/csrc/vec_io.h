// Element types and 16-byte row access of the channels-last sequence operators (norm.hip, sequence.hip).  Meant to
// be included INSIDE an anonymous namespace of the including translation unit.
#pragma once

// Longest vector a lane moves in one instruction: 16 bytes.
template <typename T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));

// A row of C elements of an odd C, or of a slice of a projection, starts at any multiple of the element size.  The
// hardware takes unaligned 16-byte global accesses (gfx950 under ROCm runs with unaligned access on), so one code
// path serves every alignment: the type below only promises the alignment of an element.
template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
    T v[V];
};

// The first n of V elements at p (n >= V: all of them in one load); the others are zero and never read.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T *p, int n) {
    Pack<T, V> r;
    if (n >= V) {
        r = *reinterpret_cast<const Pack<T, V> *>(p);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) r.v[e] = e < n ? p[e] : static_cast<T>(0.0f);
    }
    return r;
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, V> &r, int n) {
    if (n >= V) {
        *reinterpret_cast<Pack<T, V> *>(p) = r;
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < n) p[e] = r.v[e];
    }
}

__device__ __forceinline__ float silu(float x) { return x * __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

// Activation codes are SEDMI_ACT_* (sedmi.h); the code is uniform, the branch costs a scalar compare.
__device__ __forceinline__ float activate(float x, int act) {
    if (act == SEDMI_ACT_RELU) return x < 0.0f ? 0.0f : x;      // NaN stays NaN
    if (act == SEDMI_ACT_SILU) return silu(x);
    if (act == SEDMI_ACT_GELU) return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f));
    return x;
}

__device__ __forceinline__ int64_t clamp_length(const int64_t *lengths, int64_t i, int64_t most) {
    if (lengths == nullptr) return most;
    const int64_t n = lengths[i];
    return n < 0 ? 0 : (n > most ? most : n);
}

// Dispatches f(T{}) on a SEDMI_DTYPE_* code.
template <typename F>
int with_dtype(int dtype, F f) {
    if (dtype == SEDMI_DTYPE_F32) return f(float{});
    if (dtype == SEDMI_DTYPE_F16) return f(static_cast<_Float16>(0.0f));
    return f(static_cast<__bf16>(0.0f));
}
