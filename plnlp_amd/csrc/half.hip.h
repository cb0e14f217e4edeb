// 16-bit storage helpers shared by the lookup, linear_act and grad_clip kernels (gfx950, wave64).
// Every computation is in f32 (or f64): a value is widened when it is read and rounded ONCE, to nearest even, when it is stored.
#pragma once
#include "common.hip.h"

namespace plnlp {

typedef __bf16   bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float    f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

inline bool is_dtype(int d) { return d == PLNLP_DTYPE_F32 || d == PLNLP_DTYPE_BF16 || d == PLNLP_DTYPE_F16; }
inline int dtype_size(int d) { return d == PLNLP_DTYPE_F32 ? 4 : 2; }

// V consecutive elements as one access (V * sizeof(T) bytes, at most 16 per load instruction; aligned to that)
template <typename T, int V> struct alignas(V * sizeof(T) > 16 ? 16 : V * sizeof(T)) Pack { T v[V]; };

// the same at any alignment of whole elements (global memory takes it, at a part of the rate where rows straddle lines)
template <typename T, int V> struct __attribute__((packed, aligned(sizeof(T)))) LoosePack { T v[V]; };
template <typename T, int V, bool LOOSE> struct PackOf { typedef Pack<T, V> type; };
template <typename T, int V> struct PackOf<T, V, true> { typedef LoosePack<T, V> type; };

template <typename T, int V> __device__ __forceinline__ void load_f32(const T* p, float (&x)[V]) {
    const Pack<T, V> k = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = (float)k.v[i];
}
template <typename T, int V> __device__ __forceinline__ void store_f32(T* p, const float (&x)[V]) {
    Pack<T, V> k;
#pragma unroll
    for (int i = 0; i < V; ++i) k.v[i] = (T)x[i];
    *reinterpret_cast<Pack<T, V>*>(p) = k;
}

// ... past the caches, for what is larger than they are and so would only drive out what the next kernel reads
template <typename T, int V> __device__ __forceinline__ void stream_f32(T* p, const float (&x)[V]) {
    Pack<T, V> k;
#pragma unroll
    for (int i = 0; i < V; ++i) k.v[i] = (T)x[i];
    if constexpr (sizeof(k) % 16 == 0) {
        struct Quads { u32x4 q[sizeof(k) / 16]; };
        const Quads q = __builtin_bit_cast(Quads, k);
#pragma unroll
        for (unsigned i = 0; i < sizeof(k) / 16; ++i) __builtin_nontemporal_store(q.q[i], reinterpret_cast<u32x4*>(p) + i);
    } else *reinterpret_cast<Pack<T, V>*>(p) = k;
}
// a pack that is read once
template <typename T, int V> __device__ __forceinline__ Pack<T, V> stream_pack(const T* p) {
    if constexpr (sizeof(Pack<T, V>) % 16 == 0) {
        struct Quads { u32x4 q[sizeof(Pack<T, V>) / 16]; } k;
#pragma unroll
        for (unsigned i = 0; i < sizeof(k) / 16; ++i) k.q[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p) + i);
        return __builtin_bit_cast(Pack<T, V>, k);
    } else return *reinterpret_cast<const Pack<T, V>*>(p);
}
constexpr int64_t STREAM_BYTES = (int64_t)128 << 20;       // half of the Infinity Cache

// one call of f with the C++ types of a run-time dtype
template <typename F> inline int with_dtype(int d, F&& f) {
    if (d == PLNLP_DTYPE_F32) return f(float{});
    if (d == PLNLP_DTYPE_BF16) return f(__bf16{});
    return f(_Float16{});
}

}  // namespace plnlp
