// LayerNorm with the residual add before it, forward and backward (dk_net_layer_norm_*).
//
//   s = x + delta (rounded to T), mu = mean(s), r = 1 / sqrt(mean((s - mu)^2) + eps), h = (s - mu) r w + b
//   g = dh w, n = (s - mu) r:  ds = r (g - mean(g) - n mean(g n)) + ds_res,  dw = sum dh n,  db = sum dh
//
// Memory-bound (~10 operations an element forward, ~15 backward), so each pass reads its inputs once: a
// row lives in the registers of LANES threads, NV 16-byte vectors each, and both reductions (the
// variance is of differences from the mean, not of squares) run on the registers.  (Above 12288 columns the
// backward pass has 12 to 38 registers too few a thread, which go to scratch memory.)
//   With the residual add, forward / backward (a copy reaches 4.6 TB/s): 31744 x 256 f32 28 us, 4.7 TB/s /
// 24 us, 5.4 TB/s, and 4 us for the join; 16384 x 4096 bf16 99 us, 5.4 TB/s / 117 us, 4.6 TB/s, and 8 us.
// Rows of odd width in 16 bits begin between dwords, which costs the cache 20 to 40 %: 50030 x 1111 f16 61 us
// forward against 51 at 1104 columns, 117 against 85 backward.  Wide rows, with the residual add: 4096 x 12288 f32 169 /
// 167 us, 4.8 TB/s, bf16 89 / 100, 4.5 and 4.0; 4096 x 16384 f32 220 / 239, 4.9 and 4.5, bf16 123 / 142, 4.4 and 3.8.
#pragma once
#include "train_common.h"

namespace dk {
namespace train {

// The threads that share a row and the vectors that each holds.  Groups of 8 lanes read 128 bytes side
// by side, a cache line; a row's group grows where a thread would hold more than 16 elements, and, to
// stay within one wave (no barrier), 32 at 64 lanes; 256 threads hold 16 elements each up to 4096
// columns, 512 threads 32 up to 16384.
template <int LANES_, int NV_>
struct NormShape {
    static constexpr int LANES = LANES_, NV = NV_, THREADS = LANES_ > 256 ? LANES_ : 256, ROWS = THREADS / LANES_;
    // whether column c + j of vector i lies in a row of d: only the last vector can reach behind it, as with one
    // vector less a row would not fit
    static __device__ __forceinline__ bool inside(int i, uint32_t c, uint32_t d) { return i + 1 < NV_ || c < d; }
    // whether the next row is loaded under the present one's reductions: where registers are left for it
    template <class T>
    static constexpr bool AHEAD = NV_ * VEC<T> <= 16;
};

// sums of two values over a row's threads; `buf` alternates between calls, so one barrier a call is enough
template <int LANES>
__device__ __forceinline__ void row_sum(float& a, float& b, float2 (*lds)[LANES / WAVE + 1], int buf) {
    a = lanes_reduce<(LANES < WAVE ? LANES : WAVE), Add>(a);
    b = lanes_reduce<(LANES < WAVE ? LANES : WAVE), Add>(b);
    if constexpr (LANES > WAVE) {
        if (threadIdx.x % WAVE == 0) lds[buf][threadIdx.x / WAVE] = make_float2(a, b);
        __syncthreads();
        a = b = 0.0f;
#pragma unroll
        for (int i = 0; i < LANES / WAVE; ++i) {
            a += lds[buf][i].x;
            b += lds[buf][i].y;
        }
    }
}

// NV vectors of a weight (f32 or T) as f32; `none` where there is no weight
template <class T, int NV, int LANES>
__device__ __forceinline__ void load_weight(const void* w, bool f32, float none, uint32_t t, uint32_t d, float (*out)[VEC<T>]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t c = (t + i * LANES) * VEC<T>;
        if (!w) {
#pragma unroll
            for (int j = 0; j < VEC<T>; ++j) out[i][j] = none;
        } else if (f32) {
#pragma unroll
            for (int q = 0; q < VEC<T> / 4; ++q) {
                const Vec<float> v = load_vec((const float*)w, c + 4 * q, d);
#pragma unroll
                for (int j = 0; j < 4; ++j) out[i][4 * q + j] = v[j];
            }
        } else {
            const Vec<T> v = load_vec((const T*)w, c, d);
#pragma unroll
            for (int j = 0; j < VEC<T>; ++j) out[i][j] = to_f32((T)v[j]);
        }
    }
}

struct NormArgs {
    const void *x, *delta;
    uint64_t xs, ds, rows;
    uint32_t d;
    bool wf32;
    const void *w, *b;
    float eps, inv_d;
    void *x_out, *h;
    float* stats;
};

template <class T, int NV, int LANES>
__device__ __forceinline__ void load_row(const void* base, uint64_t stride, uint64_t row, uint32_t t, uint32_t d, Vec<T>* out) {
    const T* x = (const T*)base + row * stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) out[i] = load_vec(x, (t + i * LANES) * VEC<T>, d);
}

template <class T, class S>
__global__ __launch_bounds__(S::THREADS) void layer_norm_kernel(NormArgs a) {
    constexpr int L = S::LANES, NV = S::NV, V = VEC<T>;
    __shared__ float2 lds[2][L / WAVE + 1];
    const uint32_t t = threadIdx.x % L, d = a.d;
    const uint64_t step = (uint64_t)gridDim.x * S::ROWS, last = a.rows - 1;
    uint64_t row = (uint64_t)blockIdx.x * S::ROWS + threadIdx.x / L;   // (a group behind the last row repeats that one, without storing)
    Vec<T> raw[NV], add[NV];
    auto load = [&](uint64_t at) {
        at = at < last ? at : last;
        load_row<T, NV, L>(a.x, a.xs, at, t, d, raw);
        if (a.delta) load_row<T, NV, L>(a.delta, a.ds, at, t, d, add);
    };
    if (S::template AHEAD<T>) load(row);
    float w[NV][V], b[NV][V];
    load_weight<T, NV, L>(a.w, a.wf32, 1.0f, t, d, w);
    load_weight<T, NV, L>(a.b, a.wf32, 0.0f, t, d, b);
    for (uint64_t base = (uint64_t)blockIdx.x * S::ROWS; base < a.rows; base += step, row += step) {
        const bool live = row < a.rows;
        if (!S::template AHEAD<T>) load(row);
        float v[NV][V];
        float sum = 0.0f, none = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (a.delta) raw[i][j] = from_f32<T>(to_f32((T)raw[i][j]) + to_f32((T)add[i][j]));
                v[i][j] = to_f32((T)raw[i][j]);
                sum += v[i][j];
            }
        if (a.x_out && live) {
            T* s = (T*)a.x_out + row * d;
#pragma unroll
            for (int i = 0; i < NV; ++i) store_vec(s, (t + i * L) * V, d, raw[i]);
        }
        if (S::template AHEAD<T> && base + step < a.rows) load(row + step);
        row_sum<L>(sum, none, lds, 0);
        const float mu = sum / (float)d;   // (a quotient: the mean of equal values is that value)
        float sq = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[i][j] = S::inside(i, (t + i * L) * V + j, d) ? v[i][j] - mu : 0.0f;
                sq += v[i][j] * v[i][j];
            }
        row_sum<L>(sq, none, lds, 1);
        const float r = 1.0f / sqrtf(sq * a.inv_d + a.eps);
        if (!live) continue;
        T* h = (T*)a.h + row * d;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            Vec<T> o;
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = from_f32<T>(v[i][j] * r * w[i][j] + b[i][j]);
            store_vec(h, (t + i * L) * V, d, o);
        }
        if (a.stats && t == 0) *(float2*)(a.stats + 2 * row) = make_float2(mu, r);
    }
}

struct NormBwdArgs {
    const void *dh, *dres, *x;
    uint64_t dhs, drs, xs, rows;
    uint32_t d;
    bool wf32;
    const float* stats;
    const void* w;
    float inv_d;
    void* dx;
    float* part;   // [gridDim.x][2][d] partial sums of dw and db, or NULL
};

// One pass: dx, and each workgroup's share of dw and db in registers (a thread keeps its columns over all
// its rows), joined over the workgroup's rows in LDS at the end.
template <class T, class S>
__global__ __launch_bounds__(S::THREADS) void layer_norm_bwd_kernel(NormBwdArgs a) {
    constexpr int L = S::LANES, NV = S::NV, V = VEC<T>;
    __shared__ float2 lds[2][L / WAVE + 1];
    const uint32_t t = threadIdx.x % L, d = a.d;
    float w[NV][V], aw[NV][V], ab[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) aw[i][j] = ab[i][j] = 0.0f;
    int buf = 0;
    const uint64_t step = (uint64_t)gridDim.x * S::ROWS, last = a.rows - 1;
    uint64_t row = (uint64_t)blockIdx.x * S::ROWS + threadIdx.x / L;
    Vec<T> xr[NV], gr[NV], res[NV];
    float2 st;
    auto load = [&](uint64_t at) {   // (0 behind the row's end)
        at = at < last ? at : last;
        st = *(const float2*)(a.stats + 2 * at);
        load_row<T, NV, L>(a.x, a.xs, at, t, d, xr);
        load_row<T, NV, L>(a.dh, a.dhs, at, t, d, gr);
        if (a.dres) load_row<T, NV, L>(a.dres, a.drs, at, t, d, res);
    };
    if (S::template AHEAD<T>) load(row);
    load_weight<T, NV, L>(a.w, a.wf32, 1.0f, t, d, w);
    for (uint64_t base = (uint64_t)blockIdx.x * S::ROWS; base < a.rows; base += step, row += step) {
        const bool live = row < a.rows;
        if (!S::template AHEAD<T>) load(row);
        const float mu = st.x, r = st.y;
        float sg = 0.0f, sgn = 0.0f, n[NV][V], g[NV][V], e[NV][V];
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float g0 = live ? to_f32((T)gr[i][j]) : 0.0f;
                n[i][j] = S::inside(i, (t + i * L) * V + j, d) ? (to_f32((T)xr[i][j]) - mu) * r : 0.0f;
                g[i][j] = g0 * w[i][j];
                if (a.dres) e[i][j] = to_f32((T)res[i][j]);
                sg += g[i][j];
                sgn += g[i][j] * n[i][j];
                aw[i][j] += g0 * n[i][j];
                ab[i][j] += g0;
            }
        if (S::template AHEAD<T> && base + step < a.rows) load(row + step);
        row_sum<L>(sg, sgn, lds, buf);
        buf ^= 1;
        if (!live) continue;
        const float mg = sg * a.inv_d, mgn = sgn * a.inv_d;
        T* dx = (T*)a.dx + row * d;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            Vec<T> o;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float v = r * (g[i][j] - mg - n[i][j] * mgn);
                o[j] = from_f32<T>(a.dres ? v + e[i][j] : v);
            }
            store_vec(dx, (t + i * L) * V, d, o);
        }
    }
    if (!a.part) return;
    __shared__ float join[S::ROWS > 1 ? S::ROWS * L * NV * V : 1];
    float* part = a.part + (uint64_t)blockIdx.x * 2 * d;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if constexpr (S::ROWS == 1) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const uint32_t c = (t + i * L) * V + j;
                    if (c < d) part[k * d + c] = k ? ab[i][j] : aw[i][j];
                }
        } else {
            constexpr int W = L * NV * V;   // a row's columns, rounded up
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) join[(threadIdx.x / L) * W + (t + i * L) * V + j] = k ? ab[i][j] : aw[i][j];
            __syncthreads();
            for (uint32_t c = threadIdx.x; c < d; c += S::THREADS) {
                float s = 0.0f;
#pragma unroll
                for (int q = 0; q < S::ROWS; ++q) s += join[q * W + c];
                part[k * d + c] = s;
            }
        }
    }
}

// the workgroups' shares of dw and db: 16 columns x 64 threads, each over every 64th share, then a tree
template <class W>
__global__ __launch_bounds__(1024) void layer_norm_dw_join_kernel(const float* part, uint32_t parts, uint32_t d, W* dw, W* db) {
    __shared__ float lds[64][17];
    const uint32_t tx = threadIdx.x % 16, ty = threadIdx.x / 16, i = blockIdx.x * 16 + tx;
    float s = 0.0f;
    if (i < 2 * d)
#pragma unroll 8
        for (uint32_t k = ty; k < parts; k += 64) s += part[(uint64_t)k * 2 * d + i];
    lds[ty][tx] = s;
    __syncthreads();
    s = wave_sum(lds[threadIdx.x % 64][threadIdx.x / 64]);   // (transposed: a wave sums a column)
    const uint32_t o = blockIdx.x * 16 + threadIdx.x / 64;
    if (threadIdx.x % 64 != 0 || o >= 2 * d) return;
    W* out = o < d ? dw : db;
    if (out) out[o < d ? o : o - d] = from_f32<W>(s);
}

}  // namespace train
}  // namespace dk
