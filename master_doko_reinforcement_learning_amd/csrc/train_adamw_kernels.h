// An AdamW step over many tensors at once (dk_net_adamw_async).
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Moments in f32, or in 8 bits: e4m3 codes of m and of sqrt(v) (the root halves v's range of exponents)
// with one f32 scale, largest magnitude / 448, for each block of 256 elements.  A positive root is kept
// at e4m3's least value at least: rounded to zero, the element's next step would be m / eps.  The step
// itself uses the moments before they are rounded.
//
// Memory-bound: 28 bytes an element in f32, 16 with 8-bit states, against ~30 operations.  64 M bf16 weights with
// f32 masters take 342 us, 5.5 TB/s; 63 M f32 weights with 8-bit states 174 us, 5.8 TB/s (202 us with
// single elements a lane); a network's 99 tensors, 3.2 M weights, 18 us and 3 us for the tick.
#pragma once
#include "train_common.h"

namespace dk {
namespace train {

constexpr uint32_t ADAMW_BLOCK = 256;     // elements of a wave: 4 a lane; a block of 8-bit states
constexpr uint32_t ADAMW_TENSORS = 104;   // of a launch: they go in its arguments, up to 4 KB of them
constexpr uint32_t ADAMW_TICKS = 960;

struct AdamwTable {
    void* p[ADAMW_TENSORS];
    const void* g[ADAMW_TENSORS];
    uint64_t n[ADAMW_TENSORS];
    uint32_t block[ADAMW_TENSORS];         // the tensor's first block of 256 in the states
    uint32_t id[ADAMW_TENSORS];            // its place in factors[]
    uint32_t first[ADAMW_TENSORS];         // its first workgroup
    uint32_t count;
};
struct AdamwTicks {
    uint32_t id[ADAMW_TICKS];
    uint32_t count;
};

// t += 1 and the step's factors of every tensor listed: lr / (1 - b1^t), 1 / sqrt(1 - b2^t) and
// 1 - lr wd.  On the device, so that a captured step counts its replays.
__global__ __launch_bounds__(64) void adamw_tick_kernel(AdamwTicks tick, double lr, const float* d_lr, double log_b1, double log_b2,
                                                        double wd, int32_t* step, float* factors) {
    const uint32_t i = blockIdx.x * 64 + threadIdx.x;
    if (i >= tick.count) return;
    const uint32_t id = tick.id[i];
    const int32_t t = step[id] + 1;
    step[id] = t;
    if (d_lr) lr = (double)*d_lr;
    factors[3 * id] = (float)(lr / -expm1((double)t * log_b1));
    factors[3 * id + 1] = (float)(1.0 / sqrt(-expm1((double)t * log_b2)));
    factors[3 * id + 2] = (float)(1.0 - lr * wd);
}

struct AdamwArgs {
    float b1, c1, b2, c2, eps;
    void *m, *v;
    float *ms, *vs, *master;
    const float* factors;
};

template <class T>
using Vec4 __attribute__((aligned(alignof(T)))) = T __attribute__((ext_vector_type(4)));

// 4 elements of a tensor, 0 behind its end (left: how many there are)
template <class T>
__device__ __forceinline__ void load4(const T* x, uint32_t left, float* out) {
    if (left >= 4) {
        const Vec4<T> v = *(const Vec4<T>*)x;
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j] = to_f32((T)v[j]);
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) out[j] = j < left ? to_f32(x[j]) : 0.0f;
    }
}
template <class T>
__device__ __forceinline__ void store4(T* x, uint32_t left, const float* in) {
    if (left >= 4) {
        Vec4<T> v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = from_f32<T>(in[j]);
        *(Vec4<T>*)x = v;
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
            if (j < left) x[j] = from_f32<T>(in[j]);
    }
}
// 4 e4m3 codes in a word, and back
__device__ __forceinline__ void codes_to_f32(uint32_t w, float* out) {
    out[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
    out[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
    out[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
    out[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
}
__device__ __forceinline__ uint32_t f32_to_codes(const float* in) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(in[0], in[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(in[2], in[3], w, true);
    return (uint32_t)w;
}
// the scale of a block of codes from its largest magnitude, and what its values are multiplied by
struct CodeScale { float scale, inverse; };
__device__ __forceinline__ CodeScale code_scale(float most) {
#pragma clang fp contract(off)
    most = wave_max(most);
    most = most < 1e-30f ? 0.0f : most;
    return {most * (1.0f / 448.0f), most > 0.0f ? 1.0f / most * 448.0f : 0.0f};
}

// A wave per block of 256 elements, 4 side by side per lane, 4 waves a workgroup.  No products are fused
// into sums and the roots and quotients are IEEE's: next to a border between two codes an element then
// takes the code that the formulas give in plain f32, whatever computes them.
template <class T, int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(AdamwTable tab, AdamwArgs a) {
#pragma clang fp contract(off)
    uint32_t k = 0;   // the last tensor that begins at or before this workgroup
    for (uint32_t half = 64; half > 0; half >>= 1)
        if (k + half < tab.count && blockIdx.x >= tab.first[k + half]) k += half;
    const uint64_t block = (uint64_t)(blockIdx.x - tab.first[k]) * 4 + threadIdx.x / WAVE;   // within the tensor
    const uint32_t lane = threadIdx.x % WAVE;
    const uint64_t at = block * ADAMW_BLOCK + 4 * lane, n = tab.n[k];
    if (block * ADAMW_BLOCK >= n) return;
    const uint32_t left = at >= n ? 0u : n - at < 4 ? (uint32_t)(n - at) : 4u;
    const uint64_t sblock = tab.block[k] + block, q = sblock * ADAMW_BLOCK + 4 * lane;
    T* p = (T*)tab.p[k] + at;
    float g[4], w[4], m[4], v[4], r[4];
    load4((const T*)tab.g[k] + at, left, g);
    if (a.master) load4(a.master + q, left, w);
    else load4(p, left, w);
    if constexpr (BITS == 8) {   // (whole words: a tensor's last block is its own to the end)
        const float ms = a.ms[sblock], vs = a.vs[sblock];
        codes_to_f32(((const uint32_t*)a.m)[q / 4], m);
        codes_to_f32(((const uint32_t*)a.v)[q / 4], v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m[j] *= ms;
            v[j] *= vs;
            v[j] *= v[j];
        }
    } else {
        load4((const float*)a.m + q, left, m);
        load4((const float*)a.v + q, left, v);
    }
    const float* f = a.factors + 3 * tab.id[k];
    const float size = f[0], iroot = f[1], keep = f[2];
    float mm = 0.0f, mr = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        m[j] = m[j] * a.b1 + g[j] * a.c1;
        v[j] = v[j] * a.b2 + g[j] * g[j] * a.c2;
        r[j] = sqrtf(v[j]);
        w[j] = w[j] * keep - size * (m[j] / (r[j] * iroot + a.eps));
        mm = fmaxf(mm, fabsf(m[j]));
        mr = fmaxf(mr, r[j]);
    }
    if (a.master) store4(a.master + q, left, w);
    store4(p, left, w);
    if constexpr (BITS == 8) {
        const CodeScale sm = code_scale(mm), sr = code_scale(mr);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m[j] *= sm.inverse;
            r[j] *= sr.inverse;
            r[j] = r[j] > 0.0f ? fmaxf(r[j], 0x1p-9f) : r[j];
        }
        if (left < 4)   // what lies behind the tensor's end stays 0, also under a scale that is not finite
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
                if (j >= left) m[j] = r[j] = 0.0f;
        ((uint32_t*)a.m)[q / 4] = f32_to_codes(m);
        ((uint32_t*)a.v)[q / 4] = f32_to_codes(r);
        if (lane == 0) {
            a.ms[sblock] = sm.scale;
            a.vs[sblock] = sr.scale;
        }
    } else {
        store4((float*)a.m + q, left, m);
        store4((float*)a.v + q, left, v);
    }
}

}  // namespace train
}  // namespace dk
