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

// sum / maximum over the 64 lanes of a wave, in every lane; a fixed tree, so equal inputs give equal bits
__device__ __forceinline__ float wave_sum(float v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

}  // namespace train
}  // namespace dk
