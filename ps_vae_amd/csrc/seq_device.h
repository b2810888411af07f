// Device helpers shared by the sequence-block kernels (norm.hip, conv.hip, scan.hip): element types, guarded vector
// access, wave reductions, sequence bounds.
#pragma once
#include "psvae_internal.h"

// A row-major operand holds fp32, bf16 or fp16 elements; all arithmetic is fp32, and a value is rounded (to nearest
// even) once, where it is stored.
typedef __bf16 bf16_t;
typedef _Float16 f16_t;

static inline size_t dtype_bytes(int dtype) { return dtype == PSVAE_F32 ? 4 : 2; }
// A launch has fewer than 2^32 threads: work beyond this many workgroups of 256 goes into further launches or a loop.
constexpr int64_t MOST_BLOCKS = 1 << 23;
static inline bool dtype_known(int dtype) { return dtype == PSVAE_F32 || dtype == PSVAE_BF16 || dtype == PSVAE_F16; }

template <class T, int V> struct VecOf { typedef T type __attribute__((ext_vector_type(V))); };

// V elements, V * sizeof(T) bytes aligned
template <int V, class T> __device__ __forceinline__ void load_vec(const T* p, float (&out)[V]) {
    if constexpr (V == 1) {
        out[0] = (float)p[0];
    } else {
        const typename VecOf<T, V>::type v = *(const typename VecOf<T, V>::type*)p;
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = (float)v[i];
    }
}
template <int V, class T> __device__ __forceinline__ void store_vec(T* p, const float (&in)[V]) {
    if constexpr (V == 1) {
        p[0] = (T)in[0];
    } else {
        typename VecOf<T, V>::type v;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (T)in[i];
        *(typename VecOf<T, V>::type*)p = v;
    }
}
// `n` of V elements (the rest 0): as one vector where `vec` says that the address allows it and all are there
template <int V, class T> __device__ __forceinline__ void load_some(const T* p, int n, bool vec, float (&out)[V]) {
    if (vec && n >= V) {
        load_vec<V>(p, out);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = i < n ? (float)p[i] : 0.f;
    }
}
template <int V, class T> __device__ __forceinline__ void store_some(T* p, int n, bool vec, const float (&in)[V]) {
    if (vec && n >= V) {
        store_vec<V>(p, in);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) p[i] = (T)in[i];
    }
}

// V elements in the type they are stored in: what a prefetch loads, so that nothing waits for it before it is used.
template <class T, int V> struct Raw {
    typename VecOf<T, V>::type v;
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (V == 1) v[0] = p[0];
        else v = *(const typename VecOf<T, V>::type*)p;
    }
    __device__ __forceinline__ float operator[](int i) const { return (float)v[i]; }
};

__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// 1 / (1 + exp(-v)): off by |v| + 3 roundings, from the scaling of v
__device__ __forceinline__ float sigmoidf(float v) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.44269504088896340736f)); }

// Sequences of packed rows: offsets [S+1] in device memory, or (offsets null) S sequences of T / S rows.  Whatever the
// offsets hold, the rows a sequence is given lie in [0, T).
struct SeqBounds { int begin, end; };
__device__ __forceinline__ SeqBounds seq_bounds(const int32_t* off, int s, int S, int T) {
    if (!off) {
        const int L = T / S;
        return {s * L, s * L + L};
    }
    const int b = min(max(off[s], 0), T);
    return {b, min(max(off[s + 1], b), T)};
}

// Whether V elements at every row of a matrix can be moved as one vector
static inline bool rows_vec(const void* p, int64_t ld, int V, int dtype) {
    const size_t unit = V * dtype_bytes(dtype);
    return !p || (((uintptr_t)p) % unit == 0 && (ld * (int64_t)dtype_bytes(dtype)) % (int64_t)unit == 0);
}

// out[c] = sum over parts of partial[part][c] in a fixed order, for `columns` columns; column c belongs to (out0, taps):
// c = k * width + d with k < taps goes to out0[d * taps + k], the last `width` columns to out1.  Null outputs are skipped.
int column_sums(hipStream_t s, const float* partial, int parts, int width, int taps, float* out0, float* out1);

#define PSVAE_BY_TYPE(dtype, T, ...)                                                     \
    do {                                                                                 \
        if ((dtype) == PSVAE_F32) { using T = float; __VA_ARGS__; }                      \
        else if ((dtype) == PSVAE_BF16) { using T = bf16_t; __VA_ARGS__; }               \
        else { using T = f16_t; __VA_ARGS__; }                                           \
    } while (0)
