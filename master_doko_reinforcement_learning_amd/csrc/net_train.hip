// The training operators of include/doko_amd.h (dk_net_layer_norm_*, dk_net_token_logprobs_*,
// dk_net_adamw_async): argument checks and launches of the kernels in train_*_kernels.h.  A translation
// unit of its own, linked into libdoko_amd.so.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>

#include "../../include/doko_amd.h"
#include "train_adamw_kernels.h"
#include "train_logp_kernels.h"
#include "train_norm_kernels.h"

namespace {

using namespace dk::train;

#define DK_HIP(call)                                              \
    do {                                                          \
        hipError_t e_ = (call);                                   \
        if (e_ != hipSuccess) {                                   \
            fprintf(stderr, "doko_amd: %s failed: %s (%s:%d)\n", #call, hipGetErrorString(e_), __FILE__, __LINE__); \
            return DK_E_LAUNCH;                                   \
        }                                                         \
    } while (0)

constexpr uint32_t NORM_MAX_D = 16384;
constexpr uint64_t MAX_ROWS = 0x7FFFFFFFull;
constexpr uint64_t ADAMW_GRID = 1ull << 23;   // workgroups of a launch: 2^33 elements

bool type_ok(int t) { return t == DK_F32 || t == DK_BF16 || t == DK_F16; }

// calls f with a value of the element type `type` names
template <class F>
void with_type(int type, F f) {
    if (type == DK_F32) f(float{});
    else if (type == DK_BF16) f(__bf16{});
    else f(_Float16{});
}
// (what lies outside would overflow in f32, as the reciprocal or in sums of differences of logits)
bool temperature_ok(float t) { return t >= 1e-6f && t <= 1e30f; }
// the same for a weight: f32, or the activations' type T
template <class T, class F>
void with_weight(int wtype, F f) {
    if (wtype == DK_F32) f(float{});
    else f(T{});
}

// calls f with the NormShape that rows of d columns of T take
template <class T, int L, int LO, int HI, class F>
void with_vectors(uint32_t nv, F f) {
    if constexpr (LO == HI) f(NormShape<L, LO>{});
    else if (nv <= (uint32_t)(L * LO)) f(NormShape<L, LO>{});
    else with_vectors<T, L, LO + 1, HI>(nv, f);
}
template <class T, class F>
void with_shape(uint32_t d, F f) {
    constexpr int E16 = 16 / VEC<T>, E32 = 32 / VEC<T>, MORE = E16 / 2 + 1;   // vectors of 16 and of 32 elements
    const uint32_t nv = (d + VEC<T> - 1) / VEC<T>;
    if (nv <= 8 * E16) with_vectors<T, 8, 1, E16>(nv, f);
    else if (nv <= 16 * E16) with_vectors<T, 16, MORE, E16>(nv, f);
    else if (nv <= 32 * E16) with_vectors<T, 32, MORE, E16>(nv, f);
    else if (nv <= 64 * E32) with_vectors<T, 64, MORE, E32>(nv, f);
    else if (nv <= 256 * E16) with_vectors<T, 256, MORE, E16>(nv, f);
    else with_vectors<T, 512, MORE, E32>(nv, f);
}

// workgroups of a norm kernel with `per` rows in a workgroup at a time
constexpr uint32_t norm_grid(uint64_t rows, uint32_t per, uint32_t most) {
    const uint64_t n = (rows + per - 1) / per;
    return n == 0 ? 1u : (uint32_t)(n < most ? n : most);
}
constexpr uint32_t NORM_GRID = 2048;
// The backward pass writes 2 d sums for each workgroup, as much as a row: no more workgroups than the 256 CUs
// hold at a time by their registers (two of 256 threads: at 16384 x 4096 bf16 108 us against 129 with 1024
// workgroups and 128 with 256; at 200000 x 160 f32 102 against 115 and 156), and at least 8 rows for each
// beyond the first 256 (2000 x 4096 bf16: 27 us against 31 with 512).
template <class S>
constexpr uint32_t norm_bwd_most(uint64_t rows) { return S::THREADS > 256 || rows < 8 * 512 ? 256u : 512u; }
uint32_t norm_bwd_grid(uint64_t rows, uint32_t d, int type) {
    uint32_t n = 1;
    with_type(type, [&](auto t) {
        with_shape<decltype(t)>(d, [&](auto s) {
            using S = decltype(s);
            n = norm_grid(rows, S::ROWS, norm_bwd_most<S>(rows));
        });
    });
    return n;
}

// Calls f with the lanes of a row and the elements of each, as types, for small vocabularies: 16 lanes up to
// 64 entries (the networks' 33 and 39 classes), a wave up to 512.
template <int G_, int E_>
struct LogpShape { static constexpr int G = G_, E = E_; };
template <class F>
void with_small_vocab(uint32_t vocab, F f) {
    if (vocab <= 16) f(LogpShape<16, 1>{});
    else if (vocab <= 32) f(LogpShape<16, 2>{});
    else if (vocab <= 48) f(LogpShape<16, 3>{});
    else if (vocab <= 64) f(LogpShape<16, 4>{});
    else if (vocab <= 128) f(LogpShape<64, 2>{});
    else if (vocab <= 256) f(LogpShape<64, 4>{});
    else f(LogpShape<64, 8>{});
}
// How rows are read: up to LOGP_SMALL entries in the registers of 16 or 64 lanes, unless many alternatives of
// a vocabulary worth their selection are wanted (20000 x 400 f32: 23 us against 24 for 5 of them, 56 against 25
// for 20); by a wave each up to 1024 entries (20000 x 1000 bf16: 20 us, 63 with a workgroup each), and up to LOGP_WAVE
// where the rows fill the GPU (4096 x 3000 bf16: 9 us against 14; 2048 x 20000: 32 against 24); else by a
// workgroup each, or, where the rows are too few, in parts of at least 2 vectors a thread, a workgroup each.  Up to
// a row for each CU, without alternatives, a workgroup of 16 waves takes a row up to LOGP_WIDE entries in one launch
// (1 x 20000 f32: 5.5 us against 7.4 in parts; 200 x 20000: 6.9 against 8.5; 1 x 131072: 11.9 against 7.2).
// The backward pass takes parts of 4 vectors a thread, a wave's up to LOGP_WAVE entries (20000 x 1000 bf16: 27 us
// against 49; 20000 x 8000 f32: 248 against 267), beyond that a workgroup's (20000 x 20000 bf16: 333 against 362).
constexpr uint32_t LOGP_SMALL = 512, LOGP_WAVE = 8192, LOGP_WIDE = 65536, LOGP_WIDE_ROWS = 256, LOGP_FILL = 1024,
                   LOGP_GROUPED = 16384, LOGP_GRID = 1u << 20;
bool logp_small(uint32_t vocab, uint32_t top) { return vocab <= LOGP_SMALL && (vocab <= 128 || top <= 8); }
struct LogpPlan { bool small, wave, wide; uint32_t splits, elems; };
LogpPlan logp_plan(uint64_t rows, uint32_t vocab, int type, uint32_t top) {
    if (logp_small(vocab, top)) return {true, false, false, 1u, vocab};
    const uint32_t unit = 256u * (type == DK_F32 ? 4u : 8u);   // a vector a thread
    const uint32_t units = (vocab + unit - 1) / unit;
    const bool wave = vocab <= 1024 || (rows >= 2048 && vocab <= LOGP_WAVE);
    if (top == 0 && !wave && rows <= LOGP_WIDE_ROWS && vocab <= LOGP_WIDE) return {false, false, true, 1u, units * unit};
    if (wave || rows >= LOGP_FILL) return {false, wave, false, 1u, units * unit};
    const uint64_t want = LOGP_FILL / (rows ? rows : 1);
    uint32_t each = (uint32_t)((units + want - 1) / want);
    each = each < 2 ? 2 : each;
    return {false, false, false, (units + each - 1) / each, each * unit};
}
uint32_t logp_grid(uint64_t jobs) { return (uint32_t)(jobs < LOGP_GRID ? jobs : LOGP_GRID); }

}  // namespace

extern "C" {

int dk_net_layer_norm_async(const void* x, uint64_t x_stride, const void* delta, uint64_t delta_stride, uint64_t rows,
                            uint32_t d, int type, const void* gamma, const void* beta, int wtype, float eps, void* x_out,
                            void* h_out, float* stats, void* stream) {
    if (!type_ok(type) || (wtype != DK_F32 && wtype != type) || d == 0 || d > NORM_MAX_D || (delta && !x_out) ||
        rows > MAX_ROWS)
        return DK_E_INVALID;
    if (rows == 0) return DK_OK;
    if (!x || !h_out) return DK_E_INVALID;
    // (x_out over rows of another pitch would overwrite some before they are read)
    if (x_out && rows > 1 && ((x_out == x && x_stride != d) || (x_out == delta && delta_stride != d))) return DK_E_INVALID;
    const NormArgs a{x, delta, x_stride, delta_stride, rows, d, wtype == DK_F32, gamma, beta, eps, 1.0f / (float)d, x_out, h_out, stats};
    with_type(type, [&](auto t) {
        using T = decltype(t);
        with_shape<T>(d, [&](auto s) {
            using S = decltype(s);
            hipLaunchKernelGGL((layer_norm_kernel<T, S>), dim3(norm_grid(rows, S::ROWS, NORM_GRID)), dim3(S::THREADS), 0,
                               (hipStream_t)stream, a);
        });
    });
    DK_HIP(hipGetLastError());
    return DK_OK;
}

uint64_t dk_net_layer_norm_bwd_workspace(uint64_t rows, uint32_t d, int type) {
    if (!type_ok(type) || d == 0 || d > NORM_MAX_D) return 0;
    return (uint64_t)norm_bwd_grid(rows, d, type) * 2 * d * sizeof(float);
}

int dk_net_layer_norm_bwd_async(const void* dh, uint64_t dh_stride, const void* dx_res, uint64_t dx_res_stride, const void* x,
                                uint64_t x_stride, const float* stats, uint64_t rows, uint32_t d, int type,
                                const void* gamma, int wtype, void* dx, void* dgamma, void* dbeta, void* workspace,
                                uint64_t workspace_bytes, void* stream) {
    if (!type_ok(type) || (wtype != DK_F32 && wtype != type) || d == 0 || d > NORM_MAX_D || rows > MAX_ROWS)
        return DK_E_INVALID;
    if (rows && (!dh || !x || !stats || !dx)) return DK_E_INVALID;
    const bool weights = dgamma || dbeta;
    if (weights && (!workspace || workspace_bytes < dk_net_layer_norm_bwd_workspace(rows, d, type))) return DK_E_INVALID;
    if (rows == 0 && !weights) return DK_OK;
    hipStream_t st = (hipStream_t)stream;
    const uint32_t grid = rows ? norm_bwd_grid(rows, d, type) : 0;
    const NormBwdArgs a{dh, dx_res, x, dh_stride, dx_res_stride, x_stride, rows, d, wtype == DK_F32, stats, gamma, 1.0f / (float)d,
                        dx, weights ? (float*)workspace : nullptr};
    with_type(type, [&](auto t) {
        using T = decltype(t);
        if (rows)
            with_shape<T>(d, [&](auto s) {
                using S = decltype(s);
                hipLaunchKernelGGL((layer_norm_bwd_kernel<T, S>), dim3(grid), dim3(S::THREADS), 0, st, a);
            });
        if (weights)
            with_weight<T>(wtype, [&](auto w) {
                using W = decltype(w);
                hipLaunchKernelGGL(layer_norm_dw_join_kernel<W>, dim3((2 * d + 15) / 16), dim3(1024), 0, st,
                                   (const float*)workspace, grid, d, (W*)dgamma, (W*)dbeta);
            });
    });
    DK_HIP(hipGetLastError());
    return DK_OK;
}

int dk_net_token_logprobs_async(const void* logits, uint64_t stride, uint64_t rows, uint32_t vocab, int type,
                                const uint8_t* mask, uint64_t mask_stride, float temperature, const int64_t* tokens,
                                uint32_t n, uint32_t top, float* logprobs, float* entropy, float* stats, float* top_logprobs,
                                int64_t* top_tokens, void* workspace, uint64_t workspace_bytes, void* stream) {
    if (!type_ok(type) || vocab == 0 || vocab > 0x7FFFFFFFu || n > TOKENS_MAX || top > TOP_MAX || rows > MAX_ROWS ||
        !temperature_ok(temperature))
        return DK_E_INVALID;
    if (rows == 0) return DK_OK;
    if (!logits || (n && (!tokens || !logprobs)) || (top && (!top_logprobs || !top_tokens))) return DK_E_INVALID;
    const uint64_t need = dk_net_token_logprobs_workspace(rows, vocab, type, top);
    if (need && (!workspace || workspace_bytes < need)) return DK_E_INVALID;
    const LogpPlan plan = logp_plan(rows, vocab, type, top);
    float* part = (float*)workspace;
    const LogpArgs a{logits, stride, rows, vocab, n, top, mask, mask_stride, 1.0f / temperature, tokens, logprobs, entropy,
                     stats, top_logprobs, top_tokens, plan.splits, plan.elems, part,
                     (uint64_t*)(part + 4 * rows * plan.splits)};
    hipStream_t st = (hipStream_t)stream;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        if (plan.small) {
            with_small_vocab(vocab, [&](auto s) {
                using S = decltype(s);
                hipLaunchKernelGGL((token_logprobs_small_kernel<T, S::G, S::E>), dim3(logp_grid((rows * S::G + 255) / 256)),
                                   dim3(256), 0, st, a);
            });
            return;
        }
        const dim3 grid(logp_grid(plan.wave ? (rows + 3) / 4 : rows * plan.splits)), block(256);
        if (plan.wave && top) hipLaunchKernelGGL((token_logprobs_kernel<T, WAVE, 1>), grid, block, 0, st, a);
        else if (plan.wave) hipLaunchKernelGGL((token_logprobs_kernel<T, WAVE, 0>), grid, block, 0, st, a);
        else if (plan.wide) hipLaunchKernelGGL((token_logprobs_kernel<T, 1024, 0>), grid, dim3(1024), 0, st, a);
        else if (top && plan.elems >= LOGP_GROUPED) hipLaunchKernelGGL((token_logprobs_kernel<T, 256, 4>), grid, block, 0, st, a);
        else if (top) hipLaunchKernelGGL((token_logprobs_kernel<T, 256, 1>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((token_logprobs_kernel<T, 256, 0>), grid, block, 0, st, a);
        if (plan.splits > 1) hipLaunchKernelGGL(token_logprobs_join_kernel<T>, dim3((uint32_t)rows), dim3(256), 0, st, a);
    });
    DK_HIP(hipGetLastError());
    return DK_OK;
}

// (a row's parts: maximum, S and U of each, then their top entries; none where a workgroup takes a row)
uint64_t dk_net_token_logprobs_workspace(uint64_t rows, uint32_t vocab, int type, uint32_t top) {
    if (!type_ok(type) || rows == 0 || vocab == 0) return 0;
    const uint32_t splits = logp_plan(rows, vocab, type, top).splits;
    return splits > 1 ? rows * splits * (4 * sizeof(float) + top * sizeof(uint64_t)) : 0;
}

int dk_net_token_logprobs_bwd_async(const void* logits, uint64_t stride, uint64_t rows, uint32_t vocab, int type,
                                    const uint8_t* mask, uint64_t mask_stride, float temperature, const int64_t* tokens,
                                    uint32_t n, const float* logprobs, const float* stats, const float* entropy,
                                    const float* dlogprobs, const float* dentropy, void* dlogits, void* stream) {
    if (!type_ok(type) || vocab == 0 || vocab > 0x7FFFFFFFu || n > TOKENS_MAX || rows > MAX_ROWS ||
        !temperature_ok(temperature))
        return DK_E_INVALID;
    if (rows == 0) return DK_OK;
    if (!logits || (n && (!tokens || !logprobs)) || !stats || !entropy || !dlogits || dlogits == logits) return DK_E_INVALID;
    const bool wave = vocab <= LOGP_WAVE;
    const uint32_t unit = (wave ? 64u : 256u) * 4u * (type == DK_F32 ? 4u : 8u), parts = (vocab + unit - 1) / unit;
    const LogpBwdArgs a{logits, stride, rows, vocab, n, mask, mask_stride, 1.0f / temperature, tokens, logprobs, stats, entropy,
                        dlogprobs, dentropy, dlogits, parts};
    hipStream_t st = (hipStream_t)stream;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        if (logp_small(vocab, 0))
            with_small_vocab(vocab, [&](auto s) {
                using S = decltype(s);
                hipLaunchKernelGGL((token_logprobs_small_bwd_kernel<T, S::G, S::E>), dim3(logp_grid((rows * S::G + 255) / 256)),
                                   dim3(256), 0, st, a);
            });
        else if (wave)
            hipLaunchKernelGGL((token_logprobs_bwd_kernel<T, WAVE>), dim3(logp_grid((rows * parts + 3) / 4)), dim3(256), 0, st, a);
        else
            hipLaunchKernelGGL((token_logprobs_bwd_kernel<T, 256>), dim3(logp_grid(rows * parts)), dim3(256), 0, st, a);
    });
    DK_HIP(hipGetLastError());
    return DK_OK;
}

int dk_net_adamw_async(const dk_net_adamw_tensor* tensors, uint32_t count, int type, int state_bits, void* exp_avg,
                       void* exp_avg_sq, float* exp_avg_scale, float* exp_avg_sq_scale, float* master, int32_t* step,
                       float* factors, double lr, const float* d_lr, double beta1, double beta2, double eps,
                       double weight_decay, void* stream) {
    if (!type_ok(type) || (state_bits != 32 && state_bits != 8) || !(beta1 >= 0.0 && beta1 < 1.0) ||
        !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0))
        return DK_E_INVALID;
    if (count == 0) return DK_OK;
    if (!tensors || !exp_avg || !exp_avg_sq || !step || !factors || (state_bits == 8 && (!exp_avg_scale || !exp_avg_sq_scale)))
        return DK_E_INVALID;
    for (uint32_t i = 0; i < count; ++i)
        if ((tensors[i].n && (!tensors[i].p || !tensors[i].g)) || tensors[i].n > ADAMW_GRID * 4 * ADAMW_BLOCK ||
            tensors[i].block > 0xFFFFFFFFull || tensors[i].id > 0xFFFFFFFFull)
            return DK_E_INVALID;
    const AdamwArgs a{(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps, exp_avg, exp_avg_sq,
                      exp_avg_scale, exp_avg_sq_scale, master, factors};
    hipStream_t st = (hipStream_t)stream;
    AdamwTicks tick;
    for (uint32_t at = 0; at < count; at += tick.count) {
        tick.count = count - at < ADAMW_TICKS ? count - at : ADAMW_TICKS;
        for (uint32_t i = 0; i < tick.count; ++i) tick.id[i] = (uint32_t)tensors[at + i].id;
        hipLaunchKernelGGL(adamw_tick_kernel, dim3((tick.count + 63) / 64), dim3(64), 0, st, tick, lr, d_lr, std::log(beta1),
                           std::log(beta2), weight_decay, step, factors);
    }
    AdamwTable tab;
    for (uint32_t at = 0; at < count;) {
        uint32_t k = 0;
        uint64_t groups = 0;
        for (; k < ADAMW_TENSORS && at < count; ++k, ++at) {
            const dk_net_adamw_tensor& t = tensors[at];
            const uint64_t more = (t.n + 4 * ADAMW_BLOCK - 1) / (4 * ADAMW_BLOCK);
            if (k && groups + more > ADAMW_GRID) break;
            tab.p[k] = t.p; tab.g[k] = t.g; tab.n[k] = t.n; tab.block[k] = (uint32_t)t.block; tab.id[k] = (uint32_t)t.id;
            tab.first[k] = (uint32_t)groups;
            groups += more;
        }
        tab.count = k;
        if (groups == 0) continue;
        with_type(type, [&](auto t) {
            using T = decltype(t);
            if (state_bits == 8)
                hipLaunchKernelGGL((adamw_kernel<T, 8>), dim3((uint32_t)groups), dim3(256), 0, st, tab, a);
            else
                hipLaunchKernelGGL((adamw_kernel<T, 32>), dim3((uint32_t)groups), dim3(256), 0, st, tab, a);
        });
    }
    DK_HIP(hipGetLastError());
    return DK_OK;
}

}  // extern "C"
