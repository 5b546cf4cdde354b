// Shared by the training operators' kernels (train_*_kernels.h): element types, unaligned vector
// accesses and cross-lane reductions.  All sums and statistics are f32; a value is rounded to the
// tensors' type (round to nearest even) only where it is stored.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace dk {
namespace train {

constexpr int WAVE = 64;

template <class T>
__device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <class T>
__device__ __forceinline__ T from_f32(float v) { return (T)v; }

// 16 bytes of elements.  Rows start wherever a view puts them, so the type promises no more than an
// element's alignment: gfx950 loads and stores 16 bytes from any address in one instruction.
template <class T>
constexpr int VEC = 16 / (int)sizeof(T);
template <class T>
using Vec __attribute__((aligned(alignof(T)))) = T __attribute__((ext_vector_type(VEC<T>)));

// the elements c .. c + VEC of a row of d, 0 behind its end
template <class T>
__device__ __forceinline__ Vec<T> load_vec(const T* row, uint32_t c, uint32_t d) {
    if (c + VEC<T> <= d) return *(const Vec<T>*)(row + c);
    Vec<T> v;
#pragma unroll
    for (int j = 0; j < VEC<T>; ++j) v[j] = c + j < d ? row[c + j] : (T)0.0f;
    return v;
}
template <class T>
__device__ __forceinline__ void store_vec(T* row, uint32_t c, uint32_t d, Vec<T> v) {
    if (c + VEC<T> <= d) {
        *(Vec<T>*)(row + c) = v;
        return;
    }
#pragma unroll
    for (int j = 0; j < VEC<T>; ++j)
        if (c + j < d) row[c + j] = v[j];
}

// v of the lane that differs in one bit of its number (1, 2: quad permutes; 4, 8: mirrors, whose lane
// holds the same value once the bits below are reduced)
template <int BIT, class U>
__device__ __forceinline__ U other(U v) {
    constexpr int CTRL = BIT == 1 ? 0xB1 : BIT == 2 ? 0x4E : BIT == 4 ? 0x141 : 0x140;
    return __builtin_bit_cast(U, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
struct Add { __device__ static float of(float a, float b) { return a + b; } };
struct Max {
    __device__ static float of(float a, float b) { return fmaxf(a, b); }
    __device__ static uint32_t of(uint32_t a, uint32_t b) { return a > b ? a : b; }
};
struct Min { __device__ static uint32_t of(uint32_t a, uint32_t b) { return a < b ? a : b; } };

// sum / maximum / minimum over groups of N lanes (a power of two up to 64), in every lane of the group;
// a fixed tree, so equal inputs give equal bits.  U: float or uint32_t.
template <int N, class Op, class U>
__device__ __forceinline__ U lanes_reduce(U v) {
    if constexpr (N >= 2) v = Op::of(v, other<1>(v));
    if constexpr (N >= 4) v = Op::of(v, other<2>(v));
    if constexpr (N >= 8) v = Op::of(v, other<4>(v));
    if constexpr (N >= 16) v = Op::of(v, other<8>(v));
    if constexpr (N >= 32) {   // (rows of 16, then halves, exchanged between two copies)
        const uint32_t u = __builtin_bit_cast(uint32_t, v);
        const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        const uint32_t lo = s[0], hi = s[1];   // (of s[1] itself a bit cast would take s[0])
        v = Op::of(__builtin_bit_cast(U, lo), __builtin_bit_cast(U, hi));
    }
    if constexpr (N >= 64) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v);
        const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        const uint32_t lo = s[0], hi = s[1];
        v = Op::of(__builtin_bit_cast(U, lo), __builtin_bit_cast(U, hi));
    }
    return v;
}
__device__ __forceinline__ float wave_sum(float v) { return lanes_reduce<64, Add>(v); }
__device__ __forceinline__ float wave_max(float v) { return lanes_reduce<64, Max>(v); }

}  // namespace train
}  // namespace dk
