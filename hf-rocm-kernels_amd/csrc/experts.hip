// Around the products of an MLP of experts: which experts a token goes to (route_experts), and its experts' rows summed again (combine_experts).
// No counterpart in the reference, whose MLP is dense.
//
// route_experts.  s[t, :] = softmax or sigmoid of the logits, in fp32.  A token goes to the `top` experts with the largest logit (scores are in the same
// order) or, with a bias, the largest s + bias; those sums lie close together, so the choice is the one that 64 bits make (choose_experts).  Of equals the
// lowest index comes first.  weights[t, j] = factor * s of the j-th choice, divided by the choices' sum where that is asked for (score_of).  Then the (token, choice)
// pairs are put in the experts' order, a token in front of a later one: rows[i] is the token of pair i, places[t, j] is where pair (t, j) went, and
// offsets[e] is where expert e begins: a counting sort, without atomics on memory (those in LDS add integers), so that equal calls give equal bits.
//
// combine_experts.  out[t] = (base ? base[t] : 0) + sum_j weights[t, j] * y[places[t, j]], in fp32, in the choices' order.
#include <cfloat>
#include <climits>
#include <cmath>
#include <type_traits>

#include "grouped_gemm.h"

namespace hfrk {

struct RouteArgs {
    const void* logits;
    const float* bias;
    const uint8_t* mask;
    float* weights;
    int32_t* experts;
    int32_t* places;
    int32_t* rows;
    int32_t* offsets;
    int32_t* counts;  // workspace: every run's pairs of every expert
    int64_t stride;   // elements between rows of the logits
    int tokens, count, top, dtype, sigmoid, renormalize;
    float factor;
};

// The largest of the wave's values, the same bits in every lane: rotations within rows of 16 lanes, then the four rows.
__device__ __forceinline__ uint32_t wave_max_unsigned(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xf, 0xf, true));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xf, 0xf, true));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xf, 0xf, true));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, true));
    const uint32_t a = max((uint32_t)__builtin_amdgcn_readlane((int)x, 0), (uint32_t)__builtin_amdgcn_readlane((int)x, 16));
    return max(a, max((uint32_t)__builtin_amdgcn_readlane((int)x, 32), (uint32_t)__builtin_amdgcn_readlane((int)x, 48)));
}

// Values as unsigned integers in the same order, above zero; zero for what is never chosen: NaN and minus infinity.  Both zeros are one.
__device__ __forceinline__ uint32_t order_of(float x) {
    x += 0.0f;
    const uint32_t b = __float_as_uint(x);
    return x > -INFINITY ? b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u) : 0u;
}

__device__ __forceinline__ uint64_t order_of(double x) {
    x += 0.0;
    const uint64_t b = (uint64_t)__double_as_longlong(x);
    return x > -(double)INFINITY ? b ^ ((b >> 63) ? ~0ull : 1ull << 63) : 0ull;
}

// e^x as 2^(x log2 e) by the hardware's exponential: off by 2^-23 and by 1.5 |x| 2^-24 of itself, which is least where the result is large.
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504089f); }

__device__ __forceinline__ double wave_sum_wide(double v) {
#pragma unroll
    for (int by = 32; by; by >>= 1) v += __shfl_xor(v, by);
    return v;
}

__device__ __forceinline__ float logit_of(const RouteArgs& a, int token, int e) {
    const long at = token * a.stride + e;
    if (a.dtype == HFRK_FP32) return static_cast<const float*>(a.logits)[at];
    return a.dtype == HFRK_BF16 ? load16<HFRK_BF16>(static_cast<const uint16_t*>(a.logits)[at]) : load16<HFRK_F16>(static_cast<const uint16_t*>(a.logits)[at]);
}

// The `top` largest keys of a wave in order, choice i's expert (`id`) in lane i of `chosen` (-1: there is none).  Keys are hi or (WIDE) hi and lo as one number,
// zero for what is never chosen.  A lane sorts its own once, so that a choice looks at one value a lane, and of equal ones takes that of the lowest lane, whose experts
// have the lowest numbers.  GAPS: whether each choice, and the best one left, is further below the one in front than margin * (1 + its size), twice what 32 bits may be
// off: then sums in 64 bits choose the same.
template <int EPL, bool WIDE, bool GAPS>
__device__ __forceinline__ bool choose_largest(uint32_t (&hi)[EPL], uint32_t (&lo)[EPL], int (&id)[EPL], int top, float margin, int* chosen) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int r = 0; r < EPL; ++r)
#pragma unroll
        for (int j = r & 1; j + 1 < EPL; j += 2) {  // neighbours change places where the second is above
            const bool swap = WIDE ? ((uint64_t)hi[j + 1] << 32 | lo[j + 1]) > ((uint64_t)hi[j] << 32 | lo[j]) : hi[j + 1] > hi[j];
            auto exchange = [&](auto& p, auto& q) __attribute__((always_inline)) {
                const auto up = swap ? q : p;
                q = swap ? p : q;
                p = up;
            };
            exchange(hi[j], hi[j + 1]);
            if constexpr (WIDE) exchange(lo[j], lo[j + 1]);
            exchange(id[j], id[j + 1]);
        }
    *chosen = -1;
    bool apart = true;
    float above = INFINITY;
    for (int i = 0; i < top + (GAPS ? 1 : 0); ++i) {
        const uint32_t best = wave_max_unsigned(hi[0]);
        if (best == 0) break;  // (a key's upper half is above zero: the smallest is that of the lowest number)
        if constexpr (GAPS) {
            const float value = __uint_as_float(best ^ ((best >> 31) ? 0x80000000u : 0xffffffffu));
            apart = apart && above - value > margin * (1.0f + fabsf(value));  // (also false where it is no number)
            above = value;
        }
        uint64_t equal = __ballot(hi[0] == best);
        if constexpr (WIDE) {
            if (equal & (equal - 1)) {  // rarely: upper halves are equal
                const uint32_t low = wave_max_unsigned(hi[0] == best ? lo[0] : 0u);
                equal = __ballot(hi[0] == best && lo[0] == low);
            }
        }
        const int owner = __builtin_ctzll(equal), expert = __builtin_amdgcn_readlane(id[0], owner);
        if (!GAPS || i < top) *chosen = lane == i ? expert : *chosen;
        const bool mine = lane == owner;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            hi[j] = mine ? (j + 1 < EPL ? hi[j + 1] : 0u) : hi[j];
            if constexpr (WIDE) lo[j] = mine ? (j + 1 < EPL ? lo[j + 1] : 0u) : lo[j];
            if (j + 1 < EPL) id[j] = mine ? id[j + 1] : id[j];
        }
    }
    return apart;
}

// Twice what s + bias may be off in 32 bits, for a sum of size v as margin * (1 + |v|).  e^-y is off by (2 + y) 2^-24 of itself (exponent rounded, hardware's
// exponential within a step).  Sigmoid, 1 / (1 + e^-x): s (1 - s) times that is at most 0.6 * 2^-24, the sum 1 + e^-x adds 2^-24 s, the reciprocal 2^-23 s, s + bias
// 2^-24 |v|: below 2^-22 (1 + |v|).  Softmax: s y is at most 0.37, the sum of up to 512 positive terms along chains of up to 20 is off by 22 * 2^-24 of itself, the
// reciprocal and the product by 3 * 2^-24: below 2^-19 (1 + |v|).
__device__ __forceinline__ float margin_of(const RouteArgs& a) { return a.sigmoid ? 0x1p-21f : 0x1p-18f; }

// A choice's score, of logit l.  One below 2^-126, e^-87.3, is not what fp32 holds, and a token's choices may all be there, or with a bias far below the others.
// Where they are divided by their sum and one of them is near it (small_score), they are made up to a factor that they share (`shared`), e^-largest, the largest
// logit of the choices (of a sigmoid where that is below zero): what then leaves fp32's range is no part of the sum either.
__device__ __forceinline__ bool small_score(const RouteArgs& a, float l, float most) { return (a.sigmoid ? l : l - most) < -80.0f; }

__device__ __forceinline__ float score_of(const RouteArgs& a, float l, float most, float sum, bool shared, float largest) {
    const float e = expf(a.sigmoid ? (shared ? -fabsf(l) : -l) : l - (shared ? largest : most));
    if (!a.sigmoid) return shared ? e : e / sum;
    return (shared && l < 0.f ? expf(l - fminf(largest, 0.f)) : 1.0f) / (1.0f + e);
}

// One wave, one token; lane l has the experts EPL l ... in registers.  Choice i's expert (-1: there is none) and weight come back in lane i; what a weight needs is
// computed for the choices only.  With a bias the choice is made in 32 bits first and is what 64 give where its values lie far enough apart; the few tokens of
// which they do not are done again.  16000 tokens on 8 of 256 experts, choosing in 64 bits at once: 28 us, with this 20.6.
// AGAIN: 32 bits have left it open already.
template <int EPL, bool BIAS, bool AGAIN = false>
__device__ __forceinline__ void choose_experts(const RouteArgs& a, int experts, int token, int* chosen, float* weight) {
    const int lane = threadIdx.x & 63, first = lane * EPL;
    *chosen = -1;
    *weight = 0.f;
    if (a.mask && !a.mask[token]) return;
    // through a buffer over the token's row: no branch, so that all are requested together
    float x[EPL];
    if (a.dtype == HFRK_FP32) {
        const __amdgpu_buffer_rsrc_t row = make_rsrc(static_cast<const float*>(a.logits) + token * a.stride, (uint32_t)experts * 4u);
#pragma unroll
        for (int j = 0; j < EPL; ++j) x[j] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(row, (first + j) * 4, 0, 0));
    } else {
        const __amdgpu_buffer_rsrc_t row = make_rsrc(static_cast<const uint16_t*>(a.logits) + token * a.stride, (uint32_t)experts * 2u);
        uint16_t h[EPL];
#pragma unroll
        for (int j = 0; j < EPL; ++j) h[j] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(row, (first + j) * 2, 0, 0);
#pragma unroll
        for (int j = 0; j < EPL; ++j) x[j] = a.dtype == HFRK_BF16 ? load16<HFRK_BF16>(h[j]) : load16<HFRK_F16>(h[j]);
    }
    float bias[EPL];
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
        x[j] = first + j < experts ? x[j] : -INFINITY;
        bias[j] = BIAS ? a.bias[min(first + j, experts - 1)] : 0.f;
    }
    bool none = false;  // a logit is NaN
    float most = x[0];
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
        none |= x[j] != x[j];
        most = fmaxf(most, x[j]);
    }
    none = __ballot(none) != 0;
    float sum = 1.f, e[EPL];
    if (!a.sigmoid) {
        most = wave_max(most);
        if (most == -INFINITY) most = 0.f;
        float part = 0.f;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            e[j] = exp_of(x[j] - most);
            part += e[j];
        }
        sum = wave_sum(part);
        none |= sum != sum;  // (a plus infinity makes every score NaN; a sigmoid's is 1)
    }
    uint32_t hi[EPL], lo[EPL];
    int id[EPL];
    bool open = AGAIN;
    if constexpr (!AGAIN) {
        const float each = __builtin_amdgcn_rcpf(sum);
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            id[j] = first + j;
            lo[j] = 0u;
            if constexpr (BIAS) {
                const float s = a.sigmoid ? __builtin_amdgcn_rcpf(1.0f + exp_of(-x[j])) : e[j] * each;
                hi[j] = x[j] > -INFINITY ? order_of(s + bias[j]) : 0u;
            } else {
                hi[j] = order_of(x[j]);
            }
        }
        open = !choose_largest<EPL, false, BIAS>(hi, lo, id, a.top, margin_of(a), chosen);
    }
    if (open && BIAS) {
        double wide[EPL], whole = 0.0;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            const double y = exp(a.sigmoid ? -(double)x[j] : (double)x[j] - (double)most);  // (one exponential for both: two took the last registers of route_few_kernel)
            wide[j] = a.sigmoid ? 1.0 / (1.0 + y) : y;
            whole += wide[j];
        }
        if (!a.sigmoid) whole = wave_sum_wide(whole);
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            const double s = a.sigmoid ? wide[j] : wide[j] / whole;
            const uint64_t key = x[j] > -INFINITY ? order_of(s + (double)bias[j]) : 0;
            id[j] = first + j;
            hi[j] = (uint32_t)(key >> 32);
            lo[j] = (uint32_t)key;
        }
        choose_largest<EPL, true, false>(hi, lo, id, a.top, 0.f, chosen);
    }
    const float l = *chosen >= 0 ? logit_of(a, token, *chosen) : INFINITY;
    const bool shared = a.renormalize && __ballot(small_score(a, l, most)) != 0;
    const float largest = shared ? wave_max(*chosen >= 0 ? l : -INFINITY) : 0.f;
    if (*chosen >= 0) *weight = score_of(a, l, most, sum, shared, largest);
    if (a.renormalize) {
        const float part = wave_sum(*weight);
        if (part != 0.f) *weight = *weight / part;
    }
    *weight *= a.factor;
    if (none) *weight = NAN;
}

__device__ __forceinline__ void store_choice(const RouteArgs& a, int token, int i, int chosen, float weight) {
    const long at = (long)token * a.top + i;
    a.weights[at] = weight;
    a.experts[at] = chosen;
    if (chosen < 0) a.places[at] = -1;  // pairs that are nothing get their place here
}

// A token a wave.
template <int EPL, bool BIAS>
__global__ void __launch_bounds__(256) choose_experts_kernel(const RouteArgs a, int experts) {
    const int lane = threadIdx.x & 63, token = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (token >= a.tokens) return;
    int chosen;
    float weight;
    choose_experts<EPL, BIAS>(a, experts, token, &chosen, &weight);
    if (lane < a.top) store_choice(a, token, lane, chosen, weight);
}

template <typename T, typename OP>
__device__ __forceinline__ T row_reduce(T v, OP op) {  // over the 16 lanes of a row, every one of which gets it
    auto rotated = [](T x, auto by) __attribute__((always_inline)) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x120 + decltype(by)::value, 0xf, 0xf, true));
    };
    v = op(v, rotated(v, std::integral_constant<int, 1>{}));
    v = op(v, rotated(v, std::integral_constant<int, 2>{}));
    v = op(v, rotated(v, std::integral_constant<int, 4>{}));
    return op(v, rotated(v, std::integral_constant<int, 8>{}));
}

// Four tokens a wave, 16 lanes each: expert 16 j + lane in register j, sorted within the lane by key and, of equal keys, number.  Many tokens are bound by
// the instructions of a choice, most of which are the same for one token and for four: 16000 tokens on 8 of 256 experts 15.2 -> 10.5 us, with a bias 21.0 -> 18.9 (of
// which the tokens that are done again are the end), 4096 on 6 of 64 4.5 -> 3.9.  A single token waits longer for it.  Tokens whose choice 32 bits leave open are done again, a wave each.
template <int EPL, bool BIAS>
__global__ void __launch_bounds__(256) choose_many_kernel(const RouteArgs a, int experts) {
    const int lane = threadIdx.x & 63, in_row = lane & 15, token0 = (blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * 4, token = token0 + (lane >> 4);
    if (token0 >= a.tokens) return;
    const bool real = token < a.tokens && (!a.mask || a.mask[token]);
    auto add = [](float x, float y) { return x + y; };
    auto larger = [](float x, float y) { return fmaxf(x, y); };
    auto above = [](uint32_t x, uint32_t y) { return max(x, y); };
    float x[EPL];
    {
        // through a buffer over the wave's rows: no branch, so that all are requested together
        const int size = a.dtype == HFRK_FP32 ? 4 : 2;
        const uint32_t rows = (uint32_t)min(4, a.tokens - token0);
        const __amdgpu_buffer_rsrc_t r = make_rsrc(static_cast<const uint8_t*>(a.logits) + token0 * a.stride * size, ((rows - 1) * (uint32_t)a.stride + (uint32_t)experts) * size);
        const int at = ((lane >> 4) * (int)a.stride + in_row) * size;
        if (a.dtype == HFRK_FP32) {
#pragma unroll
            for (int j = 0; j < EPL; ++j) x[j] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, at + j * 64, 0, 0));
        } else {
            uint16_t h[EPL];
#pragma unroll
            for (int j = 0; j < EPL; ++j) h[j] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, at + j * 32, 0, 0);
#pragma unroll
            for (int j = 0; j < EPL; ++j) x[j] = a.dtype == HFRK_BF16 ? load16<HFRK_BF16>(h[j]) : load16<HFRK_F16>(h[j]);
        }
    }
    bool none = false;
    float most = -INFINITY;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
        x[j] = j * 16 + in_row < experts ? x[j] : -INFINITY;
        none |= x[j] != x[j];
        most = fmaxf(most, x[j]);
    }
    none = row_reduce(none ? 1u : 0u, above) != 0u && real;
    float sum = 1.f, e[EPL];
    if (!a.sigmoid) {
        most = row_reduce(most, larger);
        if (most == -INFINITY) most = 0.f;
        float part = 0.f;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            e[j] = exp_of(x[j] - most);
            part += e[j];
        }
        sum = row_reduce(part, add);
        none |= sum != sum && real;  // (a plus infinity makes every score NaN; a sigmoid's is 1)
    }
    uint32_t hi[EPL], lo[EPL];  // the key, and the inverse of the expert's number: as one integer the larger is chosen first
    const float each = __builtin_amdgcn_rcpf(sum);
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
        const int expert = j * 16 + in_row;
        lo[j] = ~(uint32_t)expert;
        if constexpr (BIAS) {
            const float s = a.sigmoid ? __builtin_amdgcn_rcpf(1.0f + exp_of(-x[j])) : e[j] * each;
            hi[j] = x[j] > -INFINITY ? order_of(s + a.bias[min(expert, experts - 1)]) : 0u;
        } else {
            hi[j] = order_of(x[j]);
        }
        hi[j] = real ? hi[j] : 0u;
    }
    // Batcher's merge exchange, largest first
#pragma unroll
    for (int p = 1; p < EPL; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < EPL; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < EPL && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const int u = i + j, v = i + j + k;
                        const bool swap = ((uint64_t)hi[v] << 32 | lo[v]) > ((uint64_t)hi[u] << 32 | lo[u]);
                        const uint32_t h0 = swap ? hi[v] : hi[u], h1 = swap ? hi[u] : hi[v], l0 = swap ? lo[v] : lo[u], l1 = swap ? lo[u] : lo[v];
                        hi[u] = h0;
                        hi[v] = h1;
                        lo[u] = l0;
                        lo[v] = l1;
                    }
    int chosen[2] = {-1, -1};  // choices in_row and in_row + 16
    bool apart = true;
    const float margin = margin_of(a);
    float front = INFINITY;
    for (int i = 0; i < a.top + (BIAS ? 1 : 0); ++i) {
        const uint32_t best = row_reduce(hi[0], above);
        const uint32_t number = row_reduce(hi[0] == best ? lo[0] : 0u, above);
        if constexpr (BIAS) {
            const float value = __uint_as_float(best ^ ((best >> 31) ? 0x80000000u : 0xffffffffu));
            apart = apart && (best == 0 || front - value > margin * (1.0f + fabsf(value)));  // (also false where it is no number)
            front = value;
        }
        const int expert = best ? (int)~number : -1;
        if (i < 16) chosen[0] = in_row == i ? expert : chosen[0];
        else if (i < a.top) chosen[1] = in_row == i - 16 ? expert : chosen[1];
        const bool mine = lo[0] == number && best != 0;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            hi[j] = mine ? (j + 1 < EPL ? hi[j + 1] : 0u) : hi[j];
            if (j + 1 < EPL) lo[j] = mine ? lo[j + 1] : lo[j];
        }
    }
    if (BIAS && a.top < 16) chosen[0] = in_row < a.top ? chosen[0] : -1;  // (the one beyond the last was looked at for its distance)
    float weight[2] = {0.f, 0.f}, l[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) l[c] = chosen[c] >= 0 ? logit_of(a, token, chosen[c]) : INFINITY;
    const uint64_t small = a.renormalize ? __ballot(small_score(a, fminf(l[0], l[1]), most)) : 0;
    const bool shared = (small >> (lane & 48)) & 0xffff;
    const float largest = small ? row_reduce(fmaxf(chosen[0] >= 0 ? l[0] : -INFINITY, chosen[1] >= 0 ? l[1] : -INFINITY), larger) : 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c)
        if (chosen[c] >= 0) weight[c] = score_of(a, l[c], most, sum, shared, largest);
    if (a.renormalize) {
        const float part = row_reduce(weight[0] + weight[1], add);
        if (part != 0.f) {
            weight[0] /= part;
            weight[1] /= part;
        }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        weight[c] = none ? NAN : weight[c] * a.factor;
        if (token < a.tokens && apart && in_row + 16 * c < a.top) store_choice(a, token, in_row + 16 * c, chosen[c], weight[c]);
    }
    if constexpr (BIAS) {
        for (uint64_t again = __ballot(!apart && in_row == 0 && token < a.tokens); again; again &= again - 1) {
            const int t = token0 + __builtin_ctzll(again) / 16;
            int c;
            float w;
            choose_experts<(EPL + 3) / 4, true, true>(a, experts, t, &c, &w);
            if (lane < a.top) store_choice(a, t, lane, c, w);
        }
    }
}

// The pairs in the experts' order: each of up to 128 workgroups has a run of pairs.  Each counts its run's pairs of every expert, and in a second launch adds the
// runs' counts: those in front of its own and all, which say where its pairs begin; then it deals its run out, 1024 pairs at a time, a wave finding the lanes of
// the same expert by the bits of its number.  (A workgroup an expert, each going through all pairs twice, took 50 us of 128000 pairs and 256 experts, every
// workgroup counting all pairs in LDS 21; the two launches take 4.2 and 6.5, each a few ways to memory one after the other.)
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64, kSortGroups = 128;

__global__ void __launch_bounds__(kSortThreads) count_pairs_kernel(const RouteArgs a, int experts, int run) {
    __shared__ int counts[kMaxExperts];
    const int tid = threadIdx.x, from = blockIdx.x * run, to = min(from + run, a.count);
    if (tid < kMaxExperts) counts[tid] = 0;
    __syncthreads();
    for (int i = from + tid; i < to; i += kSortThreads) {
        const int e = a.experts[i];
        if (e >= 0) atomicAdd(&counts[e], 1);  // (of integers: their order does not matter)
    }
    __syncthreads();
    if (tid < experts) a.counts[blockIdx.x * experts + tid] = counts[tid];
}

__global__ void __launch_bounds__(kSortThreads) sort_pairs_kernel(const RouteArgs a, int experts, int run) {
    __shared__ int before[kMaxExperts], all[kMaxExperts], of_wave[kSortWaves][kMaxExperts];
    __shared__ int sums[kSortWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int from = blockIdx.x * run, to = min(from + run, a.count);
    if (tid < kMaxExperts) before[tid] = all[tid] = 0;
    __syncthreads();
    {
        const int shares = kSortThreads / experts, share = tid / experts, e = tid - share * experts;  // threads that share an expert's runs
        int front = 0, behind = 0;
        if (share < shares) {
            // through a buffer, so that the runs behind the last read zero: without a rest of single loads, each a way to memory (of 125 runs' counts 8.7 -> 6.5 us)
            const __amdgpu_buffer_rsrc_t counts = make_rsrc(a.counts, gridDim.x * (uint32_t)experts * 4u);
            for (int r0 = share; r0 < (int)gridDim.x; r0 += 16 * shares) {
                int n[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) n[j] = __builtin_amdgcn_raw_buffer_load_b32(counts, ((r0 + j * shares) * experts + e) * 4, 0, 0);
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const bool in_front = r0 + j * shares < (int)blockIdx.x;
                    front += in_front ? n[j] : 0;
                    behind += in_front ? 0 : n[j];
                }
            }
            atomicAdd(&before[e], front);
            atomicAdd(&all[e], behind);
        }
    }
    __syncthreads();
    // where each expert begins, and in it this run's pairs
    const int here = tid < kMaxExperts ? before[tid] + all[tid] : 0;
    const int upto = wave_prefix_sum(here);
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int start = upto - here;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) start += w < wave ? sums[w] : 0;
    if (tid < kMaxExperts) before[tid] += start;
    if (blockIdx.x == 0 && tid <= experts) a.offsets[tid] = start;
    // rows behind the last pair (the last thread's start is all pairs that have an expert)
    __syncthreads();
    if (tid == kSortThreads - 1) sums[0] = start;
    __syncthreads();
    const int held = sums[0];
    for (int i = max(from, held) + tid; i < to; i += kSortThreads) a.rows[i] = -1;

    const int bits = 32 - __builtin_clz(experts);
    for (int chunk = from; chunk < to; chunk += kSortThreads) {
        const int i = chunk + tid;
        const int e = i < to ? a.experts[i] : -1;
        for (int x = tid; x < kSortWaves * kMaxExperts; x += kSortThreads) (&of_wave[0][0])[x] = 0;
        __syncthreads();
        uint64_t same = __ballot(e >= 0);
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot((e >> b) & 1);
            same &= (e >> b) & 1 ? set : ~set;
        }
        const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0));
        if (e >= 0 && rank == 0) of_wave[wave][e] = __builtin_popcountll(same);
        __syncthreads();
        if (tid < experts) {  // the waves' pairs of an expert one after the other
            int at = before[tid];
#pragma unroll
            for (int w = 0; w < kSortWaves; ++w) {
                const int n = of_wave[w][tid];
                of_wave[w][tid] = at;
                at += n;
            }
            before[tid] = at;
        }
        __syncthreads();
        if (e >= 0) {
            const int place = of_wave[wave][e] + rank;
            a.places[i] = place;
            a.rows[place] = i / a.top;
        }
        __syncthreads();
    }
}

// One workgroup for all: the pairs stay in LDS, and a thread per pair counts those in front of its own.
constexpr int kFewPairs = 1024;

template <int EPL, bool BIAS>
__global__ void __launch_bounds__(kSortThreads) route_few_kernel(const RouteArgs a, int experts) {
    __shared__ __align__(16) int pairs[kFewPairs];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int padded = (a.count + 3) / 4 * 4;
    for (int token = wave; token < a.tokens; token += kSortWaves) {
        int chosen;
        float weight;
        choose_experts<EPL, BIAS>(a, experts, token, &chosen, &weight);
        if (lane < a.top) {
            const int at = token * a.top + lane;
            a.weights[at] = weight;
            a.experts[at] = chosen;
            pairs[at] = chosen < 0 ? experts : chosen;
        }
    }
    if ((int)threadIdx.x >= a.count && (int)threadIdx.x < padded) pairs[threadIdx.x] = INT_MAX;
    __syncthreads();
    const int i = threadIdx.x;
    if (i < a.count) {
        const int e = pairs[i];
        int place = 0;
        for (int j = 0; j < padded; j += 4) {
            const v4i p = *reinterpret_cast<const v4i*>(pairs + j);
#pragma unroll
            for (int v = 0; v < 4; ++v) place += p[v] < e || (p[v] == e && j + v < i);
        }
        a.places[i] = e < experts ? place : -1;
        a.rows[place] = e < experts ? i / a.top : -1;
    }
    if (i <= experts) {
        int start = 0;
        for (int j = 0; j < padded; j += 4) {
            const v4i p = *reinterpret_cast<const v4i*>(pairs + j);
#pragma unroll
            for (int v = 0; v < 4; ++v) start += p[v] < i;
        }
        a.offsets[i] = start;
    }
}

static bool route_few(int tokens, int count) { return count <= kFewPairs && tokens <= 4 * kSortWaves; }

static int route_run(int count) { return ((count + kSortGroups - 1) / kSortGroups + kSortThreads - 1) / kSortThreads * kSortThreads; }

template <int EPL, bool BIAS>
static int launch_route(const RouteArgs& a, int experts, hipStream_t stream) {
    if (route_few(a.tokens, a.count)) {
        hipLaunchKernelGGL((route_few_kernel<EPL, BIAS>), dim3(1), dim3(kSortThreads), 0, stream, a, experts);
    } else {
        // four tokens a wave need more than 512 waves of them, and rows that a wave's buffer reaches
        if (EPL <= 4 && a.tokens > 2048 && a.stride < (1 << 26))
            hipLaunchKernelGGL((choose_many_kernel<EPL <= 4 ? 4 * EPL : 4, BIAS>), dim3((a.tokens + 15) / 16), dim3(256), 0, stream, a, experts);
        else
            hipLaunchKernelGGL((choose_experts_kernel<EPL, BIAS>), dim3((a.tokens + 3) / 4), dim3(256), 0, stream, a, experts);
        HFRK_HIP_TRY(hipGetLastError());
        const int run = route_run(a.count), runs = (a.count + run - 1) / run;
        hipLaunchKernelGGL(count_pairs_kernel, dim3(runs), dim3(kSortThreads), 0, stream, a, experts, run);
        HFRK_HIP_TRY(hipGetLastError());
        hipLaunchKernelGGL(sort_pairs_kernel, dim3(runs), dim3(kSortThreads), 0, stream, a, experts, run);
    }
    HFRK_HIP_TRY(hipGetLastError());
    return HFRK_SUCCESS;
}

struct CombineArgs {
    const uint16_t* y;
    const float* weights;
    const int32_t* places;
    const uint16_t* base;
    uint16_t* output;
    int tokens, top, cols, y_rows;
};

// A thread has V columns of a token; the rows of eight choices are requested together.  V = 8: rows of whole 16-byte pieces.
template <int DT, int V>
__global__ void __launch_bounds__(256) combine_experts_kernel(const CombineArgs a) {
    constexpr int kAtOnce = 8;
    const int pieces = a.cols / V, token = blockIdx.x, piece = blockIdx.y * 256 + threadIdx.x;
    if (piece >= pieces) return;
    typedef uint16_t Piece __attribute__((ext_vector_type(V)));
    auto piece_of = [&](const uint16_t* p, long row) __attribute__((always_inline)) {
        if constexpr (V == 8) return __builtin_bit_cast(Piece, reinterpret_cast<const uint4*>(p + row * a.cols)[piece]);
        else return Piece{p[row * a.cols + piece]};
    };
    float sum[V];
#pragma unroll
    for (int v = 0; v < V; ++v) sum[v] = 0.f;
    for (int j0 = 0; j0 < a.top; j0 += kAtOnce) {
        Piece y[kAtOnce];
        float weight[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            y[j] = Piece(0);
            weight[j] = 0.f;
            if (j0 + j < a.top) {
                const long pair = (long)token * a.top + j0 + j;
                const int place = a.places[pair];
                weight[j] = a.weights[pair];
                if ((uint32_t)place < (uint32_t)a.y_rows) y[j] = piece_of(a.y, place);
            }
        }
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
            if (j0 + j < a.top) {
#pragma unroll
                for (int v = 0; v < V; ++v) sum[v] += weight[j] * load16<DT>(y[j][v]);
            }
    }
    if (a.base) {
        const Piece b = piece_of(a.base, token);
#pragma unroll
        for (int v = 0; v < V; ++v) sum[v] += load16<DT>(b[v]);
    }
    Piece out;
#pragma unroll
    for (int v = 0; v < V; ++v) out[v] = store16<DT>(sum[v]);
    if constexpr (V == 8) reinterpret_cast<uint4*>(a.output + (long)token * a.cols)[piece] = __builtin_bit_cast(uint4, out);
    else a.output[(long)token * a.cols + piece] = out[0];
}

}  // namespace hfrk

extern "C" {

size_t hfrk_route_experts_workspace_bytes(int tokens, int num_experts, int top) {
    using namespace hfrk;
    if (tokens < 1 || num_experts < 1 || num_experts > kMaxExperts || top < 1 || (long)tokens * top > (1L << 28) || route_few(tokens, tokens * top)) return 0;
    const int run = route_run(tokens * top);
    return (size_t)((tokens * top + run - 1) / run) * num_experts * sizeof(int32_t);
}

int hfrk_route_experts(const hfrk_route_args* args, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace hfrk;
    if (!args) return HFRK_BAD_SHAPE;
    RouteArgs a{args->logits, args->bias, static_cast<const uint8_t*>(args->mask), args->weights, args->experts, args->places, args->rows, args->offsets,
                static_cast<int32_t*>(workspace), args->logits_stride, args->tokens, 0, args->top, args->dtype, args->sigmoid, args->renormalize, args->factor};
    const int experts = args->num_experts;
    if (a.tokens < 0 || experts < 1 || experts > kMaxExperts || a.top < 1 || a.top > HFRK_MAX_TOP || a.top > experts) return HFRK_BAD_SHAPE;
    if (a.tokens > (1 << 24) || (long)a.tokens * a.top > (1L << 28) || a.stride < 0) return HFRK_BAD_SHAPE;
    if (a.dtype != HFRK_F16 && a.dtype != HFRK_BF16 && a.dtype != HFRK_FP32) return HFRK_BAD_DTYPE;
    if (!a.offsets || (a.tokens && (!a.logits || !a.weights || !a.experts || !a.places || !a.rows))) return HFRK_BAD_SHAPE;
    if ((reinterpret_cast<uintptr_t>(a.bias) | reinterpret_cast<uintptr_t>(a.weights) | reinterpret_cast<uintptr_t>(a.experts) |
         reinterpret_cast<uintptr_t>(a.places) | reinterpret_cast<uintptr_t>(a.rows) | reinterpret_cast<uintptr_t>(a.offsets)) & 3 ||
        reinterpret_cast<uintptr_t>(a.logits) & (a.dtype == HFRK_FP32 ? 3 : 1))
        return HFRK_BAD_ALIGNMENT;
    if (workspace_bytes < hfrk_route_experts_workspace_bytes(a.tokens, experts, a.top) || (!workspace && workspace_bytes)) return HFRK_EXCEEDS_SCRATCH;
    if (reinterpret_cast<uintptr_t>(workspace) & 3) return HFRK_BAD_ALIGNMENT;
    a.count = a.tokens * a.top;
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto with = [&](auto epl) {
        return a.bias ? launch_route<decltype(epl)::value, true>(a, experts, s) : launch_route<decltype(epl)::value, false>(a, experts, s);
    };
    if (experts <= 64) return with(std::integral_constant<int, 1>{});
    if (experts <= 128) return with(std::integral_constant<int, 2>{});
    if (experts <= 256) return with(std::integral_constant<int, 4>{});
    return with(std::integral_constant<int, 8>{});
}

int hfrk_combine_experts(const void* y, const float* weights, const int32_t* places, const void* base, void* output, int tokens, int top, int cols, int y_rows,
                         int dtype, void* stream) {
    using namespace hfrk;
    if (tokens < 0 || top < 1 || top > HFRK_MAX_TOP || cols < 1 || cols > (1 << 21) || y_rows < 0) return HFRK_BAD_SHAPE;
    if (dtype != HFRK_F16 && dtype != HFRK_BF16) return HFRK_BAD_DTYPE;
    if (tokens == 0) return HFRK_SUCCESS;
    if (tokens >= (1 << 24) || (!y && y_rows > 0) || !weights || !places || !output) return HFRK_BAD_SHAPE;
    if ((reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(places)) & 3) return HFRK_BAD_ALIGNMENT;
    const uintptr_t rows16 = reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(base) | reinterpret_cast<uintptr_t>(output);
    if (rows16 & 1) return HFRK_BAD_ALIGNMENT;
    const CombineArgs a{static_cast<const uint16_t*>(y), weights, places, static_cast<const uint16_t*>(base), static_cast<uint16_t*>(output), tokens, top, cols,
                        y_rows};
    const bool wide = cols % 8 == 0 && (rows16 & 15) == 0;
    const dim3 grid(tokens, ((wide ? cols / 8 : cols) + 255) / 256);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == HFRK_BF16) {
        if (wide) hipLaunchKernelGGL((combine_experts_kernel<HFRK_BF16, 8>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((combine_experts_kernel<HFRK_BF16, 1>), grid, dim3(256), 0, s, a);
    } else {
        if (wide) hipLaunchKernelGGL((combine_experts_kernel<HFRK_F16, 8>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((combine_experts_kernel<HFRK_F16, 1>), grid, dim3(256), 0, s, a);
    }
    HFRK_HIP_TRY(hipGetLastError());
    return HFRK_SUCCESS;
}

}  // extern "C"
