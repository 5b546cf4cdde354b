// Log probabilities of given tokens, with entropy and top alternatives, and their gradient
// (dk_net_token_logprobs_*).
//
//   z = x / T over the allowed entries; m = max z, S = sum e^(z - m), U = sum (z - m) e^(z - m)
//   lse = m + log S,  logp_i = z[t_i] - lse,  H = log S - U / S   (both terms >= 0: no cancellation)
//   dx_j = (sum_i g_i ([t_i = j] - p_j) - gH p_j (log p_j + H)) / T
//
// An entry that is masked or -inf has probability 0 and takes no gradient, whatever it holds.  The top
// alternatives are ordered by (logit descending, index ascending), compared as stored, before any
// rounding of a log probability could make ties.
#pragma once
#include "train_common.h"

namespace dk {
namespace train {

constexpr float NEG_INF = -__builtin_huge_valf();
constexpr uint32_t TOP_MAX = 32, TOKENS_MAX = 64;

// a logit's order as an unsigned key: larger key = larger value, +0 and -0 the same; 0 for what is
// never chosen (masked, -inf, NaN)
__device__ __forceinline__ uint32_t order_key(float v) {
    if (!(v > NEG_INF)) return 0u;
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t order_key(float v, uint32_t index) {
    const uint32_t k = order_key(v);
    return k ? ((uint64_t)k << 32 | (uint32_t)~index) : 0ull;
}

__device__ __forceinline__ uint64_t block_max_u64(uint64_t v, uint64_t* lds) {
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t w = __shfl_xor((unsigned long long)v, o);
        v = w > v ? w : v;
    }
    __syncthreads();
    if (threadIdx.x % WAVE == 0) lds[threadIdx.x / WAVE] = v;
    __syncthreads();
    uint64_t m = lds[0];
    for (uint32_t i = 1; i < blockDim.x / WAVE; ++i) m = lds[i] > m ? lds[i] : m;
    return m;
}
__device__ __forceinline__ float block_sum(float v, float* lds) {
    v = wave_sum(v);
    __syncthreads();
    if (threadIdx.x % WAVE == 0) lds[threadIdx.x / WAVE] = v;
    __syncthreads();
    float s = 0.0f;
    for (uint32_t i = 0; i < blockDim.x / WAVE; ++i) s += lds[i];
    return s;
}
__device__ __forceinline__ float block_max(float v, float* lds) {
    v = wave_max(v);
    __syncthreads();
    if (threadIdx.x % WAVE == 0) lds[threadIdx.x / WAVE] = v;
    __syncthreads();
    float s = lds[0];
    for (uint32_t i = 1; i < blockDim.x / WAVE; ++i) s = fmaxf(s, lds[i]);
    return s;
}

struct LogpArgs {
    const void* logits;
    uint64_t stride;
    uint64_t rows;
    uint32_t vocab, n, top;
    const uint8_t* mask;
    uint64_t mask_stride;
    float inv_t;
    const int64_t* tokens;
    float *logprobs, *entropy, *lse, *top_logprobs;
    int64_t* top_tokens;
};

// one block per row
template <class T>
__global__ __launch_bounds__(256) void token_logprobs_kernel(LogpArgs a) {
    __shared__ float lf[4];
    __shared__ uint64_t lu[4];
    const uint64_t row = blockIdx.x;
    const T* x = (const T*)a.logits + row * a.stride;
    const uint8_t* mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    auto at = [&](uint32_t c) { return !mask || mask[c] ? to_f32(x[c]) : NEG_INF; };
    float m = NEG_INF, bad = 0.0f;
    for (uint32_t c = threadIdx.x; c < a.vocab; c += 256) {
        const float v = at(c);
        m = fmaxf(m, v);
        bad += v != v || v == -NEG_INF ? 1.0f : 0.0f;
    }
    m = block_max(m, lf) * a.inv_t;
    bad = block_sum(bad, lf);
    float s = 0.0f, u = 0.0f;
    if (m > NEG_INF)
        for (uint32_t c = threadIdx.x; c < a.vocab; c += 256) {
            const float z = at(c) * a.inv_t - m;
            if (z > NEG_INF) { const float e = expf(z); s += e; u += z * e; }
        }
    s = block_sum(s, lf);
    u = block_sum(u, lf);
    float lse = m > NEG_INF ? m + logf(s) : NEG_INF, ent = m > NEG_INF ? logf(s) - u / s : 0.0f;
    if (bad > 0.0f) lse = ent = __builtin_nanf("");
    if (threadIdx.x == 0) {
        if (a.lse) a.lse[row] = lse;
        if (a.entropy) a.entropy[row] = ent;
    }
    for (uint32_t i = threadIdx.x; i < a.n; i += 256) {
        const int64_t t = a.tokens[row * a.n + i];
        float v = 0.0f;
        if (t >= (int64_t)a.vocab) v = __builtin_nanf("");
        else if (t >= 0) {
            v = at((uint32_t)t);
            v = v == NEG_INF ? (lse != lse ? lse : NEG_INF) : v * a.inv_t - lse;
        }
        a.logprobs[row * a.n + i] = v;
    }
    uint64_t last = ~0ull;
    for (uint32_t k = 0; k < a.top; ++k) {
        uint64_t best = 0;
        for (uint32_t c = threadIdx.x; c < a.vocab; c += 256) {
            const uint64_t q = order_key(at(c), c);
            if (q < last && q > best) best = q;
        }
        last = block_max_u64(best, lu);
        if (threadIdx.x == 0) {
            const uint32_t c = ~(uint32_t)last;
            a.top_tokens[row * a.top + k] = last ? (int64_t)c : -1;
            a.top_logprobs[row * a.top + k] = last ? to_f32(x[c]) * a.inv_t - lse : (lse != lse ? lse : NEG_INF);
        }
    }
}

struct LogpBwdArgs {
    const void* logits;
    uint64_t stride;
    uint64_t rows;
    uint32_t vocab, n;
    const uint8_t* mask;
    uint64_t mask_stride;
    float inv_t;
    const int64_t* tokens;
    const float *lse, *entropy, *dlogp, *dent;
    void* dx;
};

// whether token t of a row takes a gradient: neither padding, out of range, masked nor -inf
template <class T>
__device__ __forceinline__ bool takes_gradient(const T* x, const uint8_t* mask, int64_t t, uint32_t vocab) {
    return t >= 0 && t < (int64_t)vocab && (!mask || mask[t]) && to_f32(x[t]) != NEG_INF;
}

// one block per row
template <class T>
__global__ __launch_bounds__(256) void token_logprobs_bwd_kernel(LogpBwdArgs a) {
    __shared__ int32_t tok[TOKENS_MAX];
    __shared__ float grad[TOKENS_MAX];
    const uint64_t row = blockIdx.x;
    const T* x = (const T*)a.logits + row * a.stride;
    const uint8_t* mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    if (threadIdx.x < a.n) {
        const int64_t t = a.tokens[row * a.n + threadIdx.x];
        const bool ok = a.dlogp && takes_gradient(x, mask, t, a.vocab);
        tok[threadIdx.x] = ok ? (int32_t)t : -1;
        grad[threadIdx.x] = ok ? a.dlogp[row * a.n + threadIdx.x] : 0.0f;
    }
    __syncthreads();
    float total = 0.0f;
    for (uint32_t i = 0; i < a.n; ++i) total += grad[i];
    const float lse = a.lse[row], ent = a.entropy[row], ge = a.dent ? a.dent[row] : 0.0f;
    for (uint32_t c = threadIdx.x; c < a.vocab; c += 256) {
        const float v = !mask || mask[c] ? to_f32(x[c]) : NEG_INF;
        float d = 0.0f;
        if (v != NEG_INF) {
            const float lp = v * a.inv_t - lse;
            d = -expf(lp) * (total + ge * (lp + ent));
            for (uint32_t i = 0; i < a.n; ++i)
                if (tok[i] == (int32_t)c) d += grad[i];
        }
        ((T*)a.dx)[row * a.vocab + c] = from_f32<T>(d * a.inv_t);
    }
}

}  // namespace train
}  // namespace dk
