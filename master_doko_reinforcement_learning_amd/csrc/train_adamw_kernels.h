// An AdamW step over many tensors at once (dk_net_adamw_async).
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Moments in f32, or in 8 bits: e4m3 codes of m and of sqrt(v) (the root halves v's range of exponents)
// with one f32 scale, largest magnitude / 448, for each block of 256 elements.  A positive root is kept
// at e4m3's least value at least: rounded to zero, the element's next step would be m / eps.  The step
// itself uses the moments before they are rounded.
#pragma once
#include "train_common.h"

namespace dk {
namespace train {

constexpr uint32_t ADAMW_TENSORS = 64, ADAMW_BLOCK = 256;

struct AdamwTable {
    void* p[ADAMW_TENSORS];
    const void* g[ADAMW_TENSORS];
    uint64_t n[ADAMW_TENSORS];
    uint64_t block[ADAMW_TENSORS];         // the tensor's first block of 256 in the states
    uint32_t id[ADAMW_TENSORS];            // its place in step[] and factors[]
    uint32_t first[ADAMW_TENSORS + 1];     // its first workgroup
    uint32_t count;
};

// t += 1 and the step's factors of every tensor of the table: lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
// and 1 - lr wd.  On the device, so that a captured step counts its replays.
__global__ void adamw_tick_kernel(AdamwTable tab, double lr, const float* d_lr, double log_b1, double log_b2, double wd,
                                  int32_t* step, float* factors) {
    const uint32_t i = threadIdx.x;
    if (i >= tab.count) return;
    const uint32_t id = tab.id[i];
    const int32_t t = step[id] + 1;
    step[id] = t;
    if (d_lr) lr = (double)*d_lr;
    factors[3 * id] = (float)(lr / -expm1((double)t * log_b1));
    factors[3 * id + 1] = (float)(1.0 / sqrt(-expm1((double)t * log_b2)));
    factors[3 * id + 2] = (float)(1.0 - lr * wd);
}

__device__ __forceinline__ float e4m3_value(uint8_t code) { return __builtin_amdgcn_cvt_f32_fp8((int)code, 0); }
__device__ __forceinline__ uint8_t e4m3_code(float v) { return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 0xFF); }

struct AdamwArgs {
    float b1, c1, b2, c2, eps;
    void *m, *v;
    float *ms, *vs, *master;
    const float* factors;
};

// a wave per block of 256 elements, 4 per lane.  No products are fused into sums and the root and the
// quotients are IEEE's: next to a border between two codes an element then takes the code that the
// formulas give in plain f32, whatever computes them.
template <class T, int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(AdamwTable tab, AdamwArgs a) {
#pragma clang fp contract(off)
    uint32_t k = 0;
    while (k + 1 < tab.count && blockIdx.x >= tab.first[k + 1]) ++k;
    const uint64_t block = (uint64_t)(blockIdx.x - tab.first[k]) * 4 + threadIdx.x / WAVE;   // within the tensor
    const uint32_t lane = threadIdx.x % WAVE;
    const uint64_t n = tab.n[k], base = block * ADAMW_BLOCK;
    if (base >= n) return;
    const uint64_t sblock = tab.block[k] + block;
    T* p = (T*)tab.p[k];
    const T* g = (const T*)tab.g[k];
    const float size = a.factors[3 * tab.id[k]], iroot = a.factors[3 * tab.id[k] + 1], keep = a.factors[3 * tab.id[k] + 2];
    float m[4], r[4], mm = 0.0f, mr = 0.0f;
    for (int j = 0; j < 4; ++j) {
        const uint64_t e = base + j * WAVE + lane, q = sblock * ADAMW_BLOCK + j * WAVE + lane;
        m[j] = r[j] = 0.0f;
        if (e >= n) continue;
        float mv, vv;
        if (BITS == 8) {
            mv = e4m3_value(((const uint8_t*)a.m)[q]) * a.ms[sblock];
            vv = e4m3_value(((const uint8_t*)a.v)[q]) * a.vs[sblock];
            vv *= vv;
        } else {
            mv = ((const float*)a.m)[q];
            vv = ((const float*)a.v)[q];
        }
        const float gv = to_f32(g[e]);
        mv = mv * a.b1 + gv * a.c1;
        vv = vv * a.b2 + gv * gv * a.c2;
        const float root = sqrtf(vv);
        float pv = a.master ? a.master[q] : to_f32(p[e]);
        pv = pv * keep - size * (mv / (root * iroot + a.eps));
        if (a.master) a.master[q] = pv;
        p[e] = from_f32<T>(pv);
        if (BITS == 32) {
            ((float*)a.m)[q] = mv;
            ((float*)a.v)[q] = vv;
        }
        m[j] = mv;
        r[j] = root;
        mm = fmaxf(mm, fabsf(mv));
        mr = fmaxf(mr, root);
    }
    if (BITS == 8) {
        mm = wave_max(mm);
        mr = wave_max(mr);
        mm = mm < 1e-30f ? 0.0f : mm;
        mr = mr < 1e-30f ? 0.0f : mr;
        const float im = mm > 0.0f ? 1.0f / mm * 448.0f : 0.0f, ir = mr > 0.0f ? 1.0f / mr * 448.0f : 0.0f;
        for (int j = 0; j < 4; ++j) {
            const uint64_t e = base + j * WAVE + lane, q = sblock * ADAMW_BLOCK + j * WAVE + lane;
            if (e >= n) continue;
            ((uint8_t*)a.m)[q] = e4m3_code(m[j] * im);
            const float root = r[j] * ir;
            ((uint8_t*)a.v)[q] = e4m3_code(root > 0.0f ? fmaxf(root, 0x1p-9f) : root);
        }
        if (lane == 0) {
            a.ms[sblock] = mm * (1.0f / 448.0f);
            a.vs[sblock] = mr * (1.0f / 448.0f);
        }
    }
}

}  // namespace train
}  // namespace dk
