// Element types of the training-step operators: fp32, fp16 and bf16 in memory, fp32 in registers.
#pragma once
#include "common.hpp"

namespace smlvm {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

template <class T> struct KindOf;
template <> struct KindOf<float> { static constexpr int value = SMLVM_F32; };
template <> struct KindOf<f16_t> { static constexpr int value = SMLVM_F16; };
template <> struct KindOf<bf16_t> { static constexpr int value = SMLVM_BF16; };

inline int kind_bytes(int kind) { return kind == SMLVM_F32 ? 4 : 2; }
inline bool kind_ok(int kind) { return kind >= SMLVM_F32 && kind <= SMLVM_BF16; }

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// T[N] <-> float[N] through 16-byte (8-byte for 4 narrow elements) accesses.  `p` is aligned to the access.
template <class T, int N>
__device__ __forceinline__ void load_vec(const T* __restrict__ p, float (&x)[N])
{
    constexpr int BYTES = N * (int)sizeof(T);
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) {
            const u32x4 raw = reinterpret_cast<const u32x4*>(p)[i];
            T t[16 / sizeof(T)];
            __builtin_memcpy(t, &raw, 16);
#pragma unroll
            for (int j = 0; j < 16 / (int)sizeof(T); ++j) x[i * (16 / sizeof(T)) + j] = (float)t[j];
        }
    } else {
        static_assert(BYTES == 8, "8 or a multiple of 16 bytes");
        const u32x2 raw = *reinterpret_cast<const u32x2*>(p);
        T t[N];
        __builtin_memcpy(t, &raw, 8);
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = (float)t[j];
    }
}

template <class T, int N>
__device__ __forceinline__ void store_vec(T* __restrict__ p, const float (&x)[N])
{
    constexpr int BYTES = N * (int)sizeof(T);
    T t[N];
#pragma unroll
    for (int j = 0; j < N; ++j) t[j] = (T)x[j];
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) {
            u32x4 raw;
            __builtin_memcpy(&raw, &t[i * (16 / sizeof(T))], 16);
            reinterpret_cast<u32x4*>(p)[i] = raw;
        }
    } else {
        static_assert(BYTES == 8, "8 or a multiple of 16 bytes");
        u32x2 raw;
        __builtin_memcpy(&raw, t, 8);
        *reinterpret_cast<u32x2*>(p) = raw;
    }
}

// A launch's threads along one axis stay below 2^32.
inline bool grid_fits(double blocks, int threads) { return blocks * threads < 4294967296.0; }

}  // namespace smlvm
