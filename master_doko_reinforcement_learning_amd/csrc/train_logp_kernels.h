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
// of them the exponential, 7 TB/s of bf16 on 256 CUs.  A mask is a byte more for each: 4096 x 65536 bf16 152 us
// forward and 283 backward against 106 and 245 without, 8000 x 8000 f32 68 and 116 against 50 and 105.
#pragma once
#include "train_common.h"

namespace dk {
namespace train {

constexpr float NEG_INF = -__builtin_huge_valf(), LOWEST = -3.40282347e+38f, LOG2E = 1.44269504088896341f;
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

// a row's token i with its logit: loaded before the sums are, so that the two dependent reads run beside them
struct Token { float v; bool pad, over; };
template <class T>
__device__ __forceinline__ Token load_token(const LogpArgs& a, uint64_t row, uint32_t i) {
    Token k{NEG_INF, false, false};
    if (i < a.n) {
        const int64_t t = a.tokens[row * a.n + i];
        k.pad = t < 0;
        k.over = t >= (int64_t)a.vocab;
        if (!k.pad && !k.over && (!a.mask || a.mask[row * a.mask_stride + t])) k.v = to_f32(((const T*)a.logits)[row * a.stride + t]);
    }
    return k;
}
__device__ __forceinline__ void finish_token(const LogpArgs& a, uint64_t row, uint32_t i, const Token& k, const RowSoft& r) {
    if (i >= a.n) return;
    const float none = r.log_s != r.log_s ? r.log_s : NEG_INF;
    a.logprobs[row * a.n + i] = k.pad ? 0.0f : k.over ? __builtin_nanf("") : k.v == NEG_INF ? none : logprob_of(k.v, r, a.inv_t);
}
__device__ __forceinline__ void finish_stats(const LogpArgs& a, uint64_t row, const RowSoft& r) {
    if (a.stats) *(float2*)(a.stats + 2 * row) = make_float2(r.m, r.log_s);
    if (a.entropy) a.entropy[row] = r.ent;
}
__device__ __forceinline__ void finish_top(const LogpArgs& a, uint64_t row, const RowSoft& r, uint32_t k, uint64_t e) {
    a.top_tokens[row * a.top + k] = e ? (int64_t)(uint32_t)~(uint32_t)e : -1;
    a.top_logprobs[row * a.top + k] = e ? logprob_of(key_value((uint32_t)(e >> 32)), r, a.inv_t) : r.log_s != r.log_s ? r.log_s : NEG_INF;
}

// Vocabularies up to 512: G lanes share a row, E elements each in registers, 256 / G rows a workgroup.
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
        constexpr int Q = TOKENS_MAX / G;
        Token token[Q];
#pragma unroll
        for (int i = 0; i < Q; ++i) token[i] = load_token<T>(a, row, lane + i * G);
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
        if (lane == 0) finish_stats(a, row, r);
#pragma unroll
        for (int i = 0; i < Q; ++i) finish_token(a, row, lane + i * G, token[i], r);
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

// W threads that share a row: a workgroup of 4 or 16 waves, or a wave of a workgroup of 4
constexpr int team_threads(int w) { return w > 256 ? w : 256; }
template <int W>
__device__ __forceinline__ void team_sync() {
    if constexpr (W > WAVE) __syncthreads();
    else {   // (a wave's LDS accesses are done in order: the compiler must keep them so)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// The k largest of a team's entries, sorted, in lds.top[0 .. k) (0 behind the last).  A thread's entries come in
// S groups, mine[s] is the largest key of a group; scan(least, push) goes through the groups whose mine is at
// least `least` and pushes the entries whose key is; best(below) is the thread's largest entry under `below`.
//   Of a wave's groups at least k have mine >= T for the k-th largest T of them, so no entry below any
// wave's T is among the k largest: the others are few, except where many are equal.  More than ROOM of them (constant
// rows, a head that is still zero) are taken one after the other, by a pass over the team's entries each: 4096 x 32000
// f32 of equal logits take 1.87 ms with 20 alternatives and 0.78 ms with 5, of random ones 0.11 and 0.10 ms; 20000 x
// 1000 bf16 with 20 252 us against 25.
template <int W, int S>
struct TopLds {
    static constexpr uint32_t ROOM = W > WAVE ? 1024 : 256;
    uint64_t e[ROOM + 8], top[TOP_MAX], best[W / WAVE];
    uint32_t least[W / WAVE], count, n_winners, winners[S * W], keys[S][W];
};
template <int W, int BITS, int S, class Scan, class Best>
__device__ __forceinline__ void team_top(uint32_t k, const uint32_t (&mine)[S], TopLds<W, S>& lds, Scan scan, Best best) {
    const uint32_t tid = threadIdx.x % W;
    uint32_t least = 0;
    for (int b = 31; b >= 32 - BITS; --b) {
        const uint32_t next = least | 1u << b;
        uint32_t n = 0;
#pragma unroll
        for (int g = 0; g < S; ++g) n += (uint32_t)__popcll(__ballot(mine[g] >= next));
        if (n >= k) least = next;
    }
    if constexpr (W > WAVE) {
        if (tid % WAVE == 0) lds.least[tid / WAVE] = least;
    }
    if (tid == 0) lds.count = 0;
    team_sync<W>();
    if constexpr (W > WAVE)
        for (int i = 0; i < W / WAVE; ++i) least = lds.least[i] > least ? lds.least[i] : least;
    if (least == 0) least = 1;
    scan(least, [&](uint32_t key, uint32_t index) {
        const uint32_t at = atomicAdd(&lds.count, 1u);   // (any order: the ranks below depend on the set alone)
        if (at < TopLds<W, S>::ROOM) lds.e[at] = entry(key, index);
    });
    team_sync<W>();
    const uint32_t count = lds.count;
    if (count <= TopLds<W, S>::ROOM) {
        if (tid < 8) lds.e[count + tid] = 0;   // (whole groups of 8 below)
        team_sync<W>();
        for (uint32_t i = tid; i < count; i += W) {
            const uint64_t e = lds.e[i];
            uint32_t rank = 0;
            for (uint32_t j = 0; j < count; j += 8)
#pragma unroll
                for (int l = 0; l < 8; ++l) rank += lds.e[j + l] > e;
            if (rank < k) lds.top[rank] = e;
        }
        for (uint32_t i = count + tid; i < k; i += W) lds.top[i] = 0;
    } else {   // more equal ones than there is room: one after the other
        uint64_t last = ~0ull;
        for (uint32_t r = 0; r < k; ++r) {
            uint64_t e = best(last);
            for (int o = 32; o > 0; o >>= 1) {
                const uint64_t w = __shfl_xor((unsigned long long)e, o);
                e = w > e ? w : e;
            }
            if constexpr (W > WAVE) {
                team_sync<W>();
                if (tid % WAVE == 0) lds.best[tid / WAVE] = e;
                team_sync<W>();
                for (int i = 0; i < W / WAVE; ++i) e = lds.best[i] > e ? lds.best[i] : e;
            }
            if (tid == 0) lds.top[r] = e;
            last = e;
        }
    }
    team_sync<W>();
}

// S and U of a team's threads together; `lds` has an entry for each wave
template <int W>
__device__ __forceinline__ Soft team_soft(Soft a, float c, Soft* lds) {
    a = lanes_soft<WAVE>(a, c);
    if constexpr (W == WAVE) return a;
    if (threadIdx.x % WAVE == 0) lds[threadIdx.x / WAVE] = a;
    __syncthreads();
    float m = lds[0].m;
    for (int i = 1; i < W / WAVE; ++i) m = fmaxf(m, lds[i].m);
    Soft r{m, 0.0f, 0.0f};
    for (int i = 0; i < W / WAVE; ++i) {
        const Soft w = rebased(lds[i], m, c);
        r.s += w.s;
        r.u += w.u;
    }
    __syncthreads();
    return r;
}

template <class T>
using MaskVec __attribute__((aligned(1))) = uint8_t __attribute__((ext_vector_type(VEC<T>)));

// VEC logits from column at on as f32, -inf for what is masked or not below hi
template <class T, bool WHOLE>
__device__ __forceinline__ void load_logits(const T* x, const uint8_t* mask, uint32_t at, uint32_t hi, float* v) {
    if (WHOLE || at + VEC<T> <= hi) {
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
        for (int j = 0; j < VEC<T>; ++j)
            v[j] = at + j < hi && (!mask || mask[at + j]) ? to_f32(x[at + j]) : NEG_INF;
    }
}

// Larger vocabularies: W threads go once through a row, or a workgroup through one of its `splits` parts
// where the rows are too few to fill the GPU, each thread with a running maximum (rebased every 16 elements:
// 4096 x 65536 bf16 takes 99 us so, 5.4 TB/s, 107 us with 32, whose registers cost waves).  The top entries
// lie with the largest of the threads' maxima, of which there is one for each of GROUPS groups of a thread's
// elements: the groups of the largest are read again.  4 groups where a workgroup reads 16384 entries or more (1500 x
// 131072 f32 with 20 alternatives: 183 us against 251 with one), else one (20000 x 9000 f16: 159 us against 178).
// Without alternatives (GROUPS 0) the kernel has half the registers: 99 us against 118.
template <class T, int W, int GROUPS>
__global__ __launch_bounds__(team_threads(W)) void token_logprobs_kernel(LogpArgs a) {
    constexpr bool TOP = GROUPS > 0;
    constexpr int V = VEC<T>, B = 16 / V, TEAMS = team_threads(W) / W;
    __shared__ Soft soft_lds[team_threads(W) / WAVE];
    __shared__ TopLds<W, TOP ? GROUPS : 1> top_lds[TEAMS];
    auto& lds = top_lds[threadIdx.x / W];
    const uint32_t tid = threadIdx.x % W;
    const float c = a.inv_t * LOG2E;
    const uint64_t jobs = a.rows * a.splits;
    for (uint64_t job = (uint64_t)blockIdx.x * TEAMS + threadIdx.x / W; job < jobs; job += (uint64_t)gridDim.x * TEAMS) {
        const uint64_t row = W == WAVE ? job : job / a.splits;
        const uint32_t part = W == WAVE ? 0 : (uint32_t)(job % a.splits);
        const T* x = (const T*)a.logits + row * a.stride;
        const uint8_t* mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
        const uint32_t lo = part * a.part_elems, hi = a.vocab - lo > a.part_elems ? lo + a.part_elems : a.vocab;
        const uint32_t rounds = (hi - lo + W * V - 1) / (W * V);   // (vectors of a thread)
        Token token{};
        if (a.splits == 1) token = load_token<T>(a, row, tid);   // (at most 64 tokens)
        Soft mine{LOWEST, 0.0f, 0.0f};
        float seen = NEG_INF;   // the largest element of the present group
        auto take = [&](const float* v, int n) {
            float most = v[0];
#pragma unroll
            for (int j = 1; j < n; ++j) most = fmaxf(most, v[j]);
            if (TOP) seen = fmaxf(seen, most);
            const float m = fmaxf(mine.m, most);
            mine = rebased(mine, m, c);
#pragma unroll
            for (int j = 0; j < n; ++j) {
                const float z = v[j] - m, e = raw_exp2(z * c);
                mine.s += e;
                mine.u += fmaxf(z, LOWEST) * e;
            }
        };
        // a thread's elements in groups of whole batches, one after the other
        constexpr uint32_t SHARE = (TOP ? GROUPS : 1) * B;
        const uint32_t group = (rounds + SHARE - 1) / SHARE * B;   // vectors of one
        uint32_t groups = 0, ahead = group;
        uint32_t first = lo;
        float v[B * V];
        for (; hi - first >= B * W * V; first += B * W * V) {
            if (TOP && GROUPS > 1) {
                if (ahead == 0) {
                    lds.keys[groups++][tid] = order_key(seen);
                    seen = NEG_INF;
                    ahead = group;
                }
                ahead -= B;
            }
#pragma unroll
            for (int i = 0; i < B; ++i) load_logits<T, true>(x, mask, first + (i * W + tid) * V, hi, v + i * V);
            take(v, B * V);
        }
        if (TOP && GROUPS > 1 && ahead == 0 && first < hi) {
            lds.keys[groups++][tid] = order_key(seen);
            seen = NEG_INF;
        }
        // the rest, less than B vectors a thread, those that there are (each load in a branch of its own: those of whole
        // vectors are in flight together, one with a mask or behind the row's end is waited for)
#pragma unroll
        for (int i = 0; i < B; ++i)
            if (first + (i * W + tid) * V < hi) load_logits<T, false>(x, mask, first + (i * W + tid) * V, hi, v + i * V);
#pragma unroll
        for (int i = 0; i < B; ++i)
            if (first + (i * W + tid) * V < hi) take(v + i * V, V);
        const Soft all = team_soft<W>(mine, c, soft_lds);
        if constexpr (TOP) {
            uint32_t key[GROUPS];
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) key[g] = (uint32_t)g < groups ? lds.keys[g][tid] : (uint32_t)g == groups ? order_key(seen) : 0u;
            team_top<W, KEY_BITS<T>>(
                a.top, key, lds,
                [&](uint32_t least, auto push) {
                    if (tid == 0) lds.n_winners = 0;
                    team_sync<W>();
#pragma unroll
                    for (int g = 0; g < GROUPS; ++g)
                        if (key[g] >= least) lds.winners[atomicAdd(&lds.n_winners, 1u)] = g * W + tid;
                    team_sync<W>();
                    const uint32_t vectors = lds.n_winners * group;
                    for (uint32_t i = tid; i < vectors; i += W) {
                        const uint32_t w = lds.winners[i / group], at = lo + ((w / W * group + i % group) * W + w % W) * V;
                        if (at >= hi) continue;
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
                        const uint32_t at = lo + (i * W + tid) * V;
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
        }
        if (a.splits == 1) {
            const RowSoft r = finish_row(all, a.inv_t);
            if (tid == 0) finish_stats(a, row, r);
            finish_token(a, row, tid, token, r);
            if (TOP && tid < a.top) finish_top(a, row, r, tid, lds.top[tid]);
        } else {
            if (tid == 0) *(float4*)(a.part + 4 * job) = make_float4(all.m, all.s, all.u, 0.0f);
            if (TOP && tid < a.top) a.part_top[job * a.top + tid] = lds.top[tid];
        }
        team_sync<W>();
    }
}

// the parts of a row together
template <class T>
__global__ __launch_bounds__(256) void token_logprobs_join_kernel(LogpArgs a) {
    __shared__ Soft soft_lds[4];
    __shared__ TopLds<256, 1> lds;
    const uint64_t row = blockIdx.x;
    const float c = a.inv_t * LOG2E;
    const uint64_t* e = a.part_top + row * a.splits * a.top;
    const uint32_t n = a.splits * a.top;
    uint32_t key[1] = {0};
    for (uint32_t i = threadIdx.x; i < n; i += 256) {
        const uint32_t k = (uint32_t)(e[i] >> 32);
        key[0] = k > key[0] ? k : key[0];
    }
    const Token token = load_token<T>(a, row, threadIdx.x);
    Soft mine{LOWEST, 0.0f, 0.0f};
    for (uint32_t i = threadIdx.x; i < a.splits; i += 256) {
        const float4 p = *(const float4*)(a.part + 4 * (row * a.splits + i));
        const float m = fmaxf(mine.m, p.x);
        const Soft s = rebased({p.x, p.y, p.z}, m, c);
        mine = rebased(mine, m, c);
        mine.s += s.s;
        mine.u += s.u;
    }
    const RowSoft r = finish_row(team_soft<256>(mine, c, soft_lds), a.inv_t);
    if (threadIdx.x == 0) finish_stats(a, row, r);
    finish_token(a, row, threadIdx.x, token, r);
    if (a.top == 0) return;
    team_top<256, KEY_BITS<T>>(
        a.top, key, lds,
        [&](uint32_t least, auto push) {
            for (uint32_t i = threadIdx.x; i < n; i += 256) {
                const uint64_t w = e[i];
                if ((uint32_t)(w >> 32) >= least) push((uint32_t)(w >> 32), ~(uint32_t)w);
            }
        },
        [&](uint64_t below) {
            uint64_t best = 0;
            for (uint32_t i = threadIdx.x; i < n; i += 256)
                if (e[i] < below && e[i] > best) best = e[i];
            return best;
        });
    if (threadIdx.x < a.top) finish_top(a, row, r, threadIdx.x, lds.top[threadIdx.x]);
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

// a row's token i and its gradient (0 and no token for padding, out of range, and what is not allowed, whose log
// probability is -inf; in a row with a NaN or +inf every one is NaN, and so is each allowed entry's gradient without
// the tokens', while a token that is not allowed could not be told from the others)
__device__ __forceinline__ float token_gradient(const LogpBwdArgs& a, uint64_t row, uint32_t i, int32_t& token) {
    const int64_t t = a.tokens[row * a.n + i];
    const bool ok = t >= 0 && t < (int64_t)a.vocab && a.logprobs[row * a.n + i] > NEG_INF;
    token = ok ? (int32_t)t : -1;
    return ok ? a.dlogp[row * a.n + i] : 0.0f;
}
// -p (sum g + gH (log p + H)) of a logit
struct RowGrad {
    float inv_t, m, log_s, total, ge, ent;
    __device__ float of(float v) const {
        const float lp = (v - m) * inv_t - log_s, p = raw_exp2(lp * LOG2E);
        // (p log p is 0 where p is: log p may have left f32 there, as with logits of the type's lowest value)
        const float d = -p * (total + ge * (p == 0.0f ? 0.0f : lp + ent));
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

// Larger vocabularies: W threads take 4 vectors each of a row.  The tokens' columns are written again at the
// end, each by the first of its equal tokens with all their gradients in order.
template <class T, int W>
__global__ __launch_bounds__(256) void token_logprobs_bwd_kernel(LogpBwdArgs a) {
    constexpr int V = VEC<T>, B = 4, TEAMS = 256 / W;
    __shared__ int32_t team_tok[TEAMS][TOKENS_MAX];
    __shared__ float team_grad[TEAMS][TOKENS_MAX];
    const uint32_t tid = threadIdx.x % W, n = a.dlogp ? a.n : 0;
    int32_t* tok = team_tok[threadIdx.x / W];
    float* grad = team_grad[threadIdx.x / W];
    const uint64_t jobs = a.rows * a.parts;
    for (uint64_t job = (uint64_t)blockIdx.x * TEAMS + threadIdx.x / W; job < jobs; job += (uint64_t)gridDim.x * TEAMS) {
        const uint64_t row = a.rows - 1 - job / a.parts;   // from the end: what the forward pass read last may still be in the cache
        const uint32_t lo = (uint32_t)(job % a.parts) * (W * V * B);
        const T* x = (const T*)a.logits + row * a.stride;
        const uint8_t* mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
        float v[B][V];
        const bool whole = lo + W * V * B <= a.vocab;
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const uint32_t at = lo + (i * W + tid) * V;
            if (whole) load_logits<T, true>(x, mask, at, a.vocab, v[i]);
            else if (at < a.vocab) load_logits<T, false>(x, mask, at, a.vocab, v[i]);
        }
        if (tid < n) grad[tid] = token_gradient(a, row, tid, tok[tid]);
        team_sync<W>();
        float total = 0.0f;
        for (uint32_t k = 0; k < n; ++k) total += grad[k];
        const RowGrad r = row_gradient(a, row, total);
        T* dx = (T*)a.dx + row * a.vocab;
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const uint32_t at = lo + (i * W + tid) * V;
            if (!whole && at >= a.vocab) continue;
            Vec<T> o;
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = from_f32<T>(r.of(v[i][j]) * a.inv_t);
            if (whole) *(Vec<T>*)(dx + at) = o;
            else store_vec(dx, at, a.vocab, o);
        }
        team_sync<W>();   // (the columns' first values are written before their last)
        if (tid < n) {
            const int32_t t = tok[tid];
            bool first = t >= 0 && (uint32_t)t >= lo && (uint32_t)t - lo < W * V * B;
            for (uint32_t k = 0; k < tid; ++k) first = first && tok[k] != t;
            if (first) {
                float d = r.of(to_f32(x[t]));
                for (uint32_t k = tid; k < n; ++k) d += tok[k] == t ? grad[k] : 0.0f;
                dx[t] = from_f32<T>(d * a.inv_t);
            }
        }
        team_sync<W>();
    }
}

}  // namespace train
}  // namespace dk
