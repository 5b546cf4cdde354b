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
//
// Bound by reading the logits (once forward, once backward): an element costs ~11 VALU slots, a quarter
// of them the exponential, 7 TB/s of bf16 on 256 CUs.
#pragma once
#include "train_common.h"

namespace dk {
namespace train {

constexpr float NEG_INF = -__builtin_huge_valf(), LOWEST = -3.40282347e+38f, LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;
constexpr uint32_t TOP_MAX = 32, TOKENS_MAX = 64;

// a logit's order as an unsigned key: larger key = larger value, +0 and -0 the same; 0 for what is
// never chosen (masked, -inf, NaN)
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);
    return !(v > NEG_INF) ? 0u : (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __builtin_bit_cast(float, (k >> 31) ? k & 0x7FFFFFFFu : ~k);
}
// (key, index) as one number: the larger value first, of equal ones the lower index; 0 where there is none
__device__ __forceinline__ uint64_t entry(uint32_t key, uint32_t index) { return key ? (uint64_t)key << 32 | (uint32_t)~index : 0ull; }
// leading bits in which the keys of a type's values can differ
template <class T>
constexpr int KEY_BITS = sizeof(T) == 4 ? 32 : 19;

struct LogpArgs {
    const void* logits;
    uint64_t stride;
    uint64_t rows;
    uint32_t vocab, n, top;
    const uint8_t* mask;
    uint64_t mask_stride;
    float inv_t;
    const int64_t* tokens;
    float *logprobs, *entropy, *stats, *top_logprobs;
    int64_t* top_tokens;
    // a row's parts, where more than one workgroup reads it
    uint32_t splits, part_elems;
    float* part;            // [rows][splits][4]: maximum, S, U
    uint64_t* part_top;     // [rows][splits][top] entries
};

// 2^x of the instruction itself: off by one step, and 0 where the result is below 2^-126 (a probability that
// small adds nothing to a sum that has a 1 in it, and gets no gradient)
__device__ __forceinline__ float raw_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// maximum, S and U of a set of logits; U in units of x, not of x / T
struct Soft { float m, s, u; };
__device__ __forceinline__ Soft rebased(Soft a, float m, float c) {   // relative to a maximum m >= a.m
    const float dm = a.m - m, f = raw_exp2(dm * c), s = a.s * f;
    return {m, s, a.u * f + fmaxf(dm, LOWEST) * s};   // (dm may be -inf, then s is 0)
}
template <int N>
__device__ __forceinline__ Soft lanes_soft(Soft a, float c) {
    a = rebased(a, lanes_reduce<N, Max>(a.m), c);
    return {a.m, lanes_reduce<N, Add>(a.s), lanes_reduce<N, Add>(a.u)};
}

// a row's results from its sums: log S and entropy (S = 0: nothing is allowed), and the tokens' log probabilities
struct RowSoft { float m, log_s, ent; };
__device__ __forceinline__ RowSoft finish_row(Soft a, float inv_t) {
    RowSoft r;
    r.m = a.m;
    r.log_s = a.s == 0.0f ? NEG_INF : logf(a.s);
    r.ent = a.s == 0.0f ? 0.0f : r.log_s - a.u * inv_t / a.s;
    return r;
}
// log probability of an allowed logit: of differences, so that a large common offset costs nothing
__device__ __forceinline__ float logprob_of(float v, const RowSoft& r, float inv_t) { return (v - r.m) * inv_t - r.log_s; }

template <class T>
__device__ __forceinline__ void finish_tokens(const LogpArgs& a, uint64_t row, const RowSoft& r, uint32_t first, uint32_t step) {
    if (first == 0) {
        if (a.stats) *(float2*)(a.stats + 2 * row) = make_float2(r.m, r.log_s);
        if (a.entropy) a.entropy[row] = r.ent;
    }
    const T* x = (const T*)a.logits + row * a.stride;
    for (uint32_t i = first; i < a.n; i += step) {
        const int64_t t = a.tokens[row * a.n + i];
        float v = 0.0f;
        if (t >= (int64_t)a.vocab) v = __builtin_nanf("");
        else if (t >= 0) {
            v = a.mask && !a.mask[row * a.mask_stride + t] ? NEG_INF : to_f32(x[t]);
            v = v != NEG_INF ? logprob_of(v, r, a.inv_t) : r.log_s != r.log_s ? r.log_s : NEG_INF;
        }
        a.logprobs[row * a.n + i] = v;
    }
}
__device__ __forceinline__ void finish_top(const LogpArgs& a, uint64_t row, const RowSoft& r, uint32_t k, uint64_t e) {
    a.top_tokens[row * a.top + k] = e ? (int64_t)(uint32_t)~(uint32_t)e : -1;
    a.top_logprobs[row * a.top + k] = e ? logprob_of(key_value((uint32_t)(e >> 32)), r, a.inv_t) : r.log_s != r.log_s ? r.log_s : NEG_INF;
}

// Vocabularies up to 1024: G lanes share a row, E elements each in registers, 256 / G rows a workgroup.
template <class T, int G, int E>
__global__ __launch_bounds__(256) void token_logprobs_small_kernel(LogpArgs a) {
    const uint32_t lane = threadIdx.x % G;
    const float c = a.inv_t * LOG2E;
    const uint64_t step = (uint64_t)gridDim.x * (256 / G);
    for (uint64_t row = (uint64_t)blockIdx.x * (256 / G) + threadIdx.x / G; row < a.rows; row += step) {
        const T* x = (const T*)a.logits + row * a.stride;
        float v[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const uint32_t at = lane + i * G;
            v[i] = at < a.vocab ? to_f32(x[at]) : NEG_INF;
        }
        if (a.mask) {
            const uint8_t* mask = a.mask + row * a.mask_stride;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const uint32_t at = lane + i * G;
                if (at < a.vocab && !mask[at]) v[i] = NEG_INF;
            }
        }
        float m = LOWEST;
#pragma unroll
        for (int i = 0; i < E; ++i) m = fmaxf(m, v[i]);
        m = lanes_reduce<G, Max>(m);
        float s = 0.0f, u = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float z = v[i] - m, e = raw_exp2(z * c);
            s += e;
            u += fmaxf(z, LOWEST) * e;
        }
        const RowSoft r = finish_row({m, lanes_reduce<G, Add>(s), lanes_reduce<G, Add>(u)}, a.inv_t);
        finish_tokens<T>(a, row, r, lane, G);
        if (a.top == 0) continue;
        uint32_t key[E];
#pragma unroll
        for (int i = 0; i < E; ++i) key[i] = order_key(v[i]);
        for (uint32_t k = 0; k < a.top; ++k) {
            uint32_t best = 0;
#pragma unroll
            for (int i = 0; i < E; ++i) best = key[i] > best ? key[i] : best;
            best = lanes_reduce<G, Max>(best);
            uint32_t at = ~0u;
#pragma unroll
            for (int i = E - 1; i >= 0; --i) at = key[i] == best ? lane + i * G : at;
            at = lanes_reduce<G, Min>(at);
#pragma unroll
            for (int i = 0; i < E; ++i) key[i] = lane + i * G == at ? 0u : key[i];
            if (lane == 0) finish_top(a, row, r, k, entry(best, at));
        }
    }
}

// The k largest of a workgroup's entries, sorted, in out[0 .. k) (0 behind the last).  `mine` is the largest
// key among a thread's entries; scan(least, push) goes through the entries of the threads whose mine is at
// least `least` and pushes those whose key is; best(below) is the thread's largest entry under `below`.
//   Of a wave's threads at least k have mine >= T for the k-th largest T of them, so no entry below any
// wave's T is among the k largest: the others are few, except where many are equal.
struct TopLds {
    static constexpr uint32_t ROOM = 1024;
    uint64_t e[ROOM];
    uint32_t least[4], count;
    uint64_t best[4];
};
template <int BITS, class Scan, class Best>
__device__ __forceinline__ void block_top(uint32_t k, uint32_t mine, TopLds& lds, uint64_t* out, Scan scan, Best best) {
    uint32_t least = 0;
    for (int b = 31; b >= 32 - BITS; --b) {
        const uint32_t next = least | 1u << b;
        if ((uint32_t)__popcll(__ballot(mine >= next)) >= k) least = next;
    }
    __syncthreads();
    if (threadIdx.x % WAVE == 0) lds.least[threadIdx.x / WAVE] = least;
    if (threadIdx.x == 0) lds.count = 0;
    __syncthreads();
    least = 1;
    for (int i = 0; i < 4; ++i) least = lds.least[i] > least ? lds.least[i] : least;
    scan(least, [&](uint32_t key, uint32_t index) {
        const uint32_t at = atomicAdd(&lds.count, 1u);   // (any order: the ranks below depend on the set alone)
        if (at < TopLds::ROOM) lds.e[at] = entry(key, index);
    });
    __syncthreads();
    const uint32_t count = lds.count;
    if (count <= TopLds::ROOM) {
        for (uint32_t i = threadIdx.x; i < count; i += 256) {
            const uint64_t e = lds.e[i];
            uint32_t rank = 0;
            for (uint32_t j = 0; j < count; ++j) rank += lds.e[j] > e;
            if (rank < k) out[rank] = e;
        }
        for (uint32_t i = count + threadIdx.x; i < k; i += 256) out[i] = 0;
    } else {   // more equal ones than there is room: one after the other
        uint64_t last = ~0ull;
        for (uint32_t r = 0; r < k; ++r) {
            uint64_t e = best(last);
            for (int o = 32; o > 0; o >>= 1) {
                const uint64_t w = __shfl_xor((unsigned long long)e, o);
                e = w > e ? w : e;
            }
            __syncthreads();
            if (threadIdx.x % WAVE == 0) lds.best[threadIdx.x / WAVE] = e;
            __syncthreads();
            for (int i = 0; i < 4; ++i) e = lds.best[i] > e ? lds.best[i] : e;
            if (threadIdx.x == 0) out[r] = e;
            last = e;
        }
    }
    __syncthreads();
}

// S and U of a workgroup's threads together; `lds` has 4 entries
__device__ __forceinline__ Soft block_soft(Soft a, float c, Soft* lds) {
    a = lanes_soft<64>(a, c);
    if (threadIdx.x % WAVE == 0) lds[threadIdx.x / WAVE] = a;
    __syncthreads();
    float m = lds[0].m;
    for (int i = 1; i < 4; ++i) m = fmaxf(m, lds[i].m);
    Soft r{m, 0.0f, 0.0f};
    for (int i = 0; i < 4; ++i) {
        const Soft w = rebased(lds[i], m, c);
        r.s += w.s;
        r.u += w.u;
    }
    __syncthreads();
    return r;
}

template <class T>
using MaskVec __attribute__((aligned(1))) = uint8_t __attribute__((ext_vector_type(VEC<T>)));

// VEC logits from column at on as f32, -inf for what is masked or behind the row's end
template <class T, bool WHOLE>
__device__ __forceinline__ void load_logits(const T* x, const uint8_t* mask, uint32_t at, uint32_t vocab, float* v) {
    if (WHOLE || at + VEC<T> <= vocab) {
        const Vec<T> raw = *(const Vec<T>*)(x + at);
#pragma unroll
        for (int j = 0; j < VEC<T>; ++j) v[j] = to_f32((T)raw[j]);
        if (mask) {
            const MaskVec<T> k = *(const MaskVec<T>*)(mask + at);
#pragma unroll
            for (int j = 0; j < VEC<T>; ++j) v[j] = k[j] ? v[j] : NEG_INF;
        }
    } else {
#pragma unroll
        for (int j = 0; j < VEC<T>; ++j) v[j] = at + j < vocab && (!mask || mask[at + j]) ? to_f32(x[at + j]) : NEG_INF;
    }
}

// Larger vocabularies: a workgroup goes once through a row, or through one of its `splits` parts where the
// rows are too few to fill the GPU, each thread with a running maximum (rebased every 4 vectors).  The top
// entries lie with the threads of the largest maxima: their elements alone are read again.
template <class T>
__global__ __launch_bounds__(256) void token_logprobs_kernel(LogpArgs a) {
    constexpr int V = VEC<T>, B = 4;
    __shared__ Soft soft_lds[4];
    __shared__ TopLds top_lds;
    __shared__ uint64_t top[TOP_MAX];
    __shared__ uint32_t winners[256], n_winners;
    const float c = a.inv_t * LOG2E;
    const uint64_t jobs = a.rows * a.splits;
    for (uint64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
        const uint64_t row = job / a.splits;
        const uint32_t part = (uint32_t)(job % a.splits);
        const T* x = (const T*)a.logits + row * a.stride;
        const uint8_t* mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
        const uint32_t lo = part * a.part_elems, hi = a.vocab - lo > a.part_elems ? lo + a.part_elems : a.vocab;
        const uint32_t rounds = (hi - lo + 256 * V - 1) / (256 * V);   // vectors of a thread
        Soft mine{LOWEST, 0.0f, 0.0f};
        auto take = [&](const float* v, int n) {
            float m = mine.m;
#pragma unroll
            for (int j = 0; j < n; ++j) m = fmaxf(m, v[j]);
            mine = rebased(mine, m, c);
#pragma unroll
            for (int j = 0; j < n; ++j) {
                const float z = v[j] - m, e = raw_exp2(z * c);
                mine.s += e;
                mine.u += fmaxf(z, LOWEST) * e;
            }
        };
        uint32_t q = 0;
        for (; (q + B) * 256 * V <= hi - lo; q += B) {
            float v[B * V];
#pragma unroll
            for (int i = 0; i < B; ++i) load_logits<T, true>(x, mask, lo + ((q + i) * 256 + threadIdx.x) * V, hi, v + i * V);
            take(v, B * V);
        }
        for (; q < rounds; ++q) {
            float v[V];
            load_logits<T, false>(x, mask, lo + (q * 256 + threadIdx.x) * V, hi, v);
            take(v, V);
        }
        const uint32_t key = mine.s == 0.0f ? 0u : order_key(mine.m);
        const Soft all = block_soft(mine, c, soft_lds);
        if (a.top)
            block_top<KEY_BITS<T>>(
                a.top, key, top_lds, top,
                [&](uint32_t least, auto push) {
                    if (threadIdx.x == 0) n_winners = 0;
                    __syncthreads();
                    if (key >= least) winners[atomicAdd(&n_winners, 1u)] = threadIdx.x;
                    __syncthreads();
                    const uint32_t vectors = n_winners * rounds;
                    for (uint32_t i = threadIdx.x; i < vectors; i += 256) {
                        const uint32_t at = lo + (i % rounds * 256 + winners[i / rounds]) * V;
                        float v[V];
                        load_logits<T, false>(x, mask, at, hi, v);
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            const uint32_t k = order_key(v[j]);
                            if (k >= least) push(k, at + j);
                        }
                    }
                },
                [&](uint64_t below) {
                    uint64_t best = 0;
                    for (uint32_t i = 0; i < rounds; ++i) {
                        const uint32_t at = lo + (i * 256 + threadIdx.x) * V;
                        float v[V];
                        load_logits<T, false>(x, mask, at, hi, v);
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            const uint64_t e = entry(order_key(v[j]), at + j);
                            if (e < below && e > best) best = e;
                        }
                    }
                    return best;
                });
        if (a.splits == 1) {
            const RowSoft r = finish_row(all, a.inv_t);
            finish_tokens<T>(a, row, r, threadIdx.x, 256);
            if (threadIdx.x < a.top) finish_top(a, row, r, threadIdx.x, top[threadIdx.x]);
        } else {
            if (threadIdx.x == 0) *(float4*)(a.part + 4 * job) = make_float4(all.m, all.s, all.u, 0.0f);
            if (threadIdx.x < a.top) a.part_top[job * a.top + threadIdx.x] = top[threadIdx.x];
        }
        __syncthreads();
    }
}

// the parts of a row together
template <class T>
__global__ __launch_bounds__(256) void token_logprobs_join_kernel(LogpArgs a) {
    __shared__ Soft soft_lds[4];
    __shared__ TopLds top_lds;
    __shared__ uint64_t top[TOP_MAX];
    const uint64_t row = blockIdx.x;
    const float c = a.inv_t * LOG2E;
    Soft mine{LOWEST, 0.0f, 0.0f};
    for (uint32_t i = threadIdx.x; i < a.splits; i += 256) {
        const float4 p = *(const float4*)(a.part + 4 * (row * a.splits + i));
        const float m = fmaxf(mine.m, p.x);
        const Soft s = rebased({p.x, p.y, p.z}, m, c);
        mine = rebased(mine, m, c);
        mine.s += s.s;
        mine.u += s.u;
    }
    const RowSoft r = finish_row(block_soft(mine, c, soft_lds), a.inv_t);
    finish_tokens<T>(a, row, r, threadIdx.x, 256);
    if (a.top == 0) return;
    const uint64_t* e = a.part_top + row * a.splits * a.top;
    const uint32_t n = a.splits * a.top;
    uint32_t key = 0;
    for (uint32_t i = threadIdx.x; i < n; i += 256) {
        const uint32_t k = (uint32_t)(e[i] >> 32);
        key = k > key ? k : key;
    }
    block_top<KEY_BITS<T>>(
        a.top, key, top_lds, top,
        [&](uint32_t least, auto push) {
            for (uint32_t i = threadIdx.x; i < n; i += 256)
                if ((uint32_t)(e[i] >> 32) >= least) push((uint32_t)(e[i] >> 32), ~(uint32_t)e[i]);
        },
        [&](uint64_t below) {
            uint64_t best = 0;
            for (uint32_t i = threadIdx.x; i < n; i += 256)
                if (e[i] < below && e[i] > best) best = e[i];
            return best;
        });
    if (threadIdx.x < a.top) finish_top(a, row, r, threadIdx.x, top[threadIdx.x]);
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
    const float *logprobs, *stats, *entropy, *dlogp, *dent;
    void* dx;
    uint32_t parts;   // of a row
};

// a row's token i and its gradient (0 and no token for padding, out of range, and what is not allowed)
__device__ __forceinline__ float token_gradient(const LogpBwdArgs& a, uint64_t row, uint32_t i, int32_t& token) {
    const int64_t t = a.tokens[row * a.n + i];
    const bool ok = t >= 0 && t < (int64_t)a.vocab && a.logprobs[row * a.n + i] != NEG_INF;
    token = ok ? (int32_t)t : -1;
    return ok ? a.dlogp[row * a.n + i] : 0.0f;
}
// -p (sum g + gH (log p + H)) of a logit
struct RowGrad {
    float inv_t, m, log_s, total, ge, ent;
    __device__ float of(float v) const {
        const float lp = (v - m) * inv_t - log_s, d = -raw_exp2(lp * LOG2E) * (total + ge * (lp + ent));
        return v == NEG_INF ? 0.0f : d;
    }
};
__device__ __forceinline__ RowGrad row_gradient(const LogpBwdArgs& a, uint64_t row, float total) {
    const float2 st = *(const float2*)(a.stats + 2 * row);
    return {a.inv_t, st.x, st.y, total, a.dent ? a.dent[row] : 0.0f, a.entropy[row]};
}

// as token_logprobs_small_kernel; every lane compares its columns with all the row's tokens
template <class T, int G, int E>
__global__ __launch_bounds__(256) void token_logprobs_small_bwd_kernel(LogpBwdArgs a) {
    constexpr int R = 256 / G;
    __shared__ int32_t tok[R][TOKENS_MAX];
    __shared__ float grad[R][TOKENS_MAX];
    const uint32_t lane = threadIdx.x % G, slot = threadIdx.x / G;
    const uint32_t n = a.dlogp ? a.n : 0;
    for (uint64_t base = (uint64_t)blockIdx.x * R; base < a.rows; base += (uint64_t)gridDim.x * R) {
        const uint64_t row = base + slot;
        const bool live = row < a.rows;
        float v[E];
        const T* x = (const T*)a.logits + row * a.stride;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const uint32_t at = lane + i * G;
            v[i] = live && at < a.vocab && (!a.mask || a.mask[row * a.mask_stride + at]) ? to_f32(x[at]) : NEG_INF;
        }
        float total = 0.0f;
        if (live)
            for (uint32_t i = lane; i < n; i += G) {
                const float g = token_gradient(a, row, i, tok[slot][i]);
                grad[slot][i] = g;
                total += g;
            }
        total = lanes_reduce<G, Add>(total);
        __syncthreads();
        if (live) {
            const RowGrad r = row_gradient(a, row, total);
            float d[E];
#pragma unroll
            for (int i = 0; i < E; ++i) d[i] = r.of(v[i]);
            for (uint32_t k = 0; k < n; ++k) {
                const int32_t t = tok[slot][k];
                const float g = grad[slot][k];
#pragma unroll
                for (int i = 0; i < E; ++i) d[i] += t == (int32_t)(lane + i * G) ? g : 0.0f;
            }
            T* dx = (T*)a.dx + row * a.vocab;
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (lane + i * G < a.vocab) dx[lane + i * G] = from_f32<T>(d[i] * a.inv_t);
        }
        __syncthreads();
    }
}

// larger vocabularies: a workgroup takes 4 vectors a thread of a row.  The tokens' columns are written
// again at the end, each by the first of its equal tokens with all their gradients in order.
template <class T>
__global__ __launch_bounds__(256) void token_logprobs_bwd_kernel(LogpBwdArgs a) {
    constexpr int V = VEC<T>, B = 4;
    __shared__ int32_t tok[TOKENS_MAX];
    __shared__ float grad[TOKENS_MAX];
    const uint32_t n = a.dlogp ? a.n : 0;
    const uint64_t jobs = a.rows * a.parts;
    for (uint64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
        const uint64_t row = job / a.parts;
        const uint32_t lo = (uint32_t)(job % a.parts) * (256 * V * B);
        const T* x = (const T*)a.logits + row * a.stride;
        const uint8_t* mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
        float v[B][V];
        const bool whole = lo + 256 * V * B <= a.vocab;
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const uint32_t at = lo + (i * 256 + threadIdx.x) * V;
            if (whole) load_logits<T, true>(x, mask, at, a.vocab, v[i]);
            else load_logits<T, false>(x, mask, at, a.vocab, v[i]);
        }
        if (threadIdx.x < n) grad[threadIdx.x] = token_gradient(a, row, threadIdx.x, tok[threadIdx.x]);
        __syncthreads();
        float total = 0.0f;
        for (uint32_t k = 0; k < n; ++k) total += grad[k];
        const RowGrad r = row_gradient(a, row, total);
        T* dx = (T*)a.dx + row * a.vocab;
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const uint32_t at = lo + (i * 256 + threadIdx.x) * V;
            Vec<T> o;
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = from_f32<T>(r.of(v[i][j]) * a.inv_t);
            if (whole) *(Vec<T>*)(dx + at) = o;
            else if (at < a.vocab) store_vec(dx, at, a.vocab, o);
        }
        __syncthreads();   // (the columns' first values are written before their last)
        if (threadIdx.x < n) {
            const int32_t t = tok[threadIdx.x];
            bool first = t >= 0 && (uint32_t)t >= lo && (uint32_t)t - lo < 256 * V * B;
            for (uint32_t k = 0; k < threadIdx.x; ++k) first = first && tok[k] != t;
            if (first) {
                float d = r.of(to_f32(x[t]));
                for (uint32_t k = threadIdx.x; k < n; ++k) d += tok[k] == t ? grad[k] : 0.0f;
                dx[t] = from_f32<T>(d * a.inv_t);
            }
        }
        __syncthreads();
    }
}

}  // namespace train
}  // namespace dk
