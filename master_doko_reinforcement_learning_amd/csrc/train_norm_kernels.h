// LayerNorm with the residual add before it, forward and backward (dk_net_layer_norm_*).
//
//   s = x + delta (rounded to T), mu = mean(s), r = 1 / sqrt(mean((s - mu)^2) + eps), h = (s - mu) r w + b
//   g = dh w, n = (s - mu) r:  ds = r (g - mean(g) - n mean(g n)) + ds_res,  dw = sum dh n,  db = sum dh
//
// Memory-bound: ~10 operations an element forward, ~15 backward.
#pragma once
#include "train_common.h"

namespace dk {
namespace train {

// one wave per row
template <class T, class W>
__global__ __launch_bounds__(256) void layer_norm_kernel(const T* x, uint64_t xs, const T* delta, uint64_t ds, uint64_t rows,
                                                         uint32_t d, const W* w, const W* b, float eps, T* x_out, T* h,
                                                         float* stats) {
    const uint32_t lane = threadIdx.x % WAVE;
    const uint64_t row = (uint64_t)blockIdx.x * (256 / WAVE) + threadIdx.x / WAVE;
    if (row >= rows) return;
    auto at = [&](uint32_t c) {
        float v = to_f32(x[row * xs + c]);
        if (delta) v = to_f32(from_f32<T>(v + to_f32(delta[row * ds + c])));
        return v;
    };
    float sum = 0.0f;
    for (uint32_t c = lane; c < d; c += WAVE) sum += at(c);
    const float mu = wave_sum(sum) / (float)d;
    float sq = 0.0f;
    for (uint32_t c = lane; c < d; c += WAVE) { const float v = at(c) - mu; sq += v * v; }
    const float r = 1.0f / sqrtf(wave_sum(sq) / (float)d + eps);
    for (uint32_t c = lane; c < d; c += WAVE) {
        const float v = at(c);
        if (x_out) x_out[row * d + c] = from_f32<T>(v);
        h[row * d + c] = from_f32<T>((v - mu) * r * (w ? to_f32(w[c]) : 1.0f) + (b ? to_f32(b[c]) : 0.0f));
    }
    if (stats && lane == 0) { stats[2 * row] = mu; stats[2 * row + 1] = r; }
}

template <class T, class W>
__global__ __launch_bounds__(256) void layer_norm_bwd_kernel(const T* dh, uint64_t dhs, const T* dres, uint64_t drs, const T* x,
                                                             uint64_t xs, const float* stats, uint64_t rows, uint32_t d,
                                                             const W* w, T* dx) {
    const uint32_t lane = threadIdx.x % WAVE;
    const uint64_t row = (uint64_t)blockIdx.x * (256 / WAVE) + threadIdx.x / WAVE;
    if (row >= rows) return;
    const float mu = stats[2 * row], r = stats[2 * row + 1];
    float a = 0.0f, c2 = 0.0f;
    for (uint32_t c = lane; c < d; c += WAVE) {
        const float g = to_f32(dh[row * dhs + c]) * (w ? to_f32(w[c]) : 1.0f);
        a += g;
        c2 += g * ((to_f32(x[row * xs + c]) - mu) * r);
    }
    a = wave_sum(a) / (float)d;
    c2 = wave_sum(c2) / (float)d;
    for (uint32_t c = lane; c < d; c += WAVE) {
        const float g = to_f32(dh[row * dhs + c]) * (w ? to_f32(w[c]) : 1.0f);
        const float n = (to_f32(x[row * xs + c]) - mu) * r;
        float v = r * (g - a - n * c2);
        if (dres) v += to_f32(dres[row * drs + c]);
        dx[row * d + c] = from_f32<T>(v);
    }
}

// partial sums of dw and db over a slice of the rows: block (64 columns) x (slice), 4 rows at a time
template <class T>
__global__ __launch_bounds__(256) void layer_norm_dw_kernel(const T* dh, uint64_t dhs, const T* x, uint64_t xs,
                                                            const float* stats, uint64_t rows, uint32_t d, uint64_t per,
                                                            float* part) {
    __shared__ float lds[2][4][64];
    const uint32_t tx = threadIdx.x % 64, ty = threadIdx.x / 64;
    const uint32_t c = blockIdx.x * 64 + tx;
    const uint64_t lo = blockIdx.y * per, hi = lo + per < rows ? lo + per : rows;
    float aw = 0.0f, ab = 0.0f;
    if (c < d)
        for (uint64_t row = lo + ty; row < hi; row += 4) {
            const float g = to_f32(dh[row * dhs + c]);
            aw += g * ((to_f32(x[row * xs + c]) - stats[2 * row]) * stats[2 * row + 1]);
            ab += g;
        }
    lds[0][ty][tx] = aw;
    lds[1][ty][tx] = ab;
    __syncthreads();
    if (ty < 2 && c < d)
        part[((uint64_t)blockIdx.y * 2 + ty) * d + c] = (lds[ty][0][tx] + lds[ty][1][tx]) + (lds[ty][2][tx] + lds[ty][3][tx]);
}

template <class W>
__global__ __launch_bounds__(256) void layer_norm_dw_join_kernel(const float* part, uint32_t parts, uint32_t d, W* dw, W* db) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= 2 * d) return;
    float s = 0.0f;
    for (uint32_t k = 0; k < parts; ++k) s += part[(uint64_t)k * 2 * d + i];
    W* out = i < d ? dw : db;
    if (out) out[i < d ? i : i - d] = from_f32<W>(s);
}

}  // namespace train
}  // namespace dk
