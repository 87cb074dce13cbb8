// Element types, vector loads and reductions of the training operators (mz_norm.hip, mz_loss.hip, mz_clip.hip).
#pragma once
#include "mz_common.h"
#include <cstdint>
#include <initializer_list>
#include <type_traits>

namespace mz {

typedef _Float16 f16;
typedef __bf16 bf16;

inline int dtype_size(int dtype) { return dtype == MZ_F32 ? 4 : dtype == MZ_F16 || dtype == MZ_BF16 ? 2 : 0; }

inline bool aligned(size_t bytes, std::initializer_list<const void*> pointers) {
    for (const void* p : pointers)
        if ((uintptr_t)p % bytes) return false;
    return true;
}

// V elements that are loaded and stored as one access, kept as they lie in memory: 16-bit elements stay two to a register
// until they are used.  Aligned like ONE element: gfx950 takes a 4-, 8- or 16-byte access at any element address, so rows of
// odd widths and views at odd offsets keep their wide accesses.
template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Vec {
    typedef typename std::conditional<sizeof(T) * V >= 4, uint32_t, uint16_t>::type Word;
    static constexpr int kWords = sizeof(T) * V / sizeof(Word);
    Word w[kWords];

    __device__ float operator[](int i) const {
        if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, w[i]);
        else if constexpr (V == 1) return (float)__builtin_bit_cast(T, w[0]);
        else if constexpr (std::is_same<T, bf16>::value) return __builtin_bit_cast(float, i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        else return (float)__builtin_bit_cast(T, (uint16_t)(w[i / 2] >> (i & 1) * 16));
    }
};

template <typename T, int V>
__device__ inline Vec<T, V> load(const T* p) {
    return *reinterpret_cast<const Vec<T, V>*>(p);
}
// 16 bytes that are not read again soon: they need not displace what the caches hold
template <typename T, int V>
__device__ inline Vec<T, V> load_streaming(const T* p) {
    static_assert(sizeof(T) * V == 16, "a whole access");
    typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));
    return __builtin_bit_cast(Vec<T, V>, __builtin_nontemporal_load(reinterpret_cast<const Words*>(p)));
}
template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Elements {
    T v[V];
};
template <typename T, int V>
__device__ inline void store(T* p, const float (&f)[V]) {
    Elements<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = (T)f[i];       // one rounding to the stored type, to nearest even
    *reinterpret_cast<Elements<T, V>*>(p) = r;
}

template <typename T>
__device__ inline T wave_sum(T v) {
#pragma unroll
    for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
    return v;
}

// Sum over a workgroup of THREADS in a fixed order; every thread gets it.  `scratch`: THREADS / 64 entries of LDS.
template <int THREADS, typename T>
__device__ inline T block_sum(T v, T* scratch) {
    v = wave_sum(v);
    if (THREADS == 64) return v;
    __syncthreads();                                    // the scratch of an earlier sum is read no more
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    T s = scratch[0];
#pragma unroll
    for (int i = 1; i < THREADS / 64; ++i) s += scratch[i];
    return s;
}

}  // namespace mz
