// Around the products of an MLP of experts: which experts a token goes to (route_experts), and its experts' rows summed again (combine_experts).
// No counterpart in the reference, whose MLP is dense.
//
// route_experts.  s[t, :] = softmax or sigmoid of the logits, in fp32.  A token goes to the `top` experts with the largest logit (scores are in the same
// order) or, with a bias, the largest s + bias; those sums lie close together, so they are made and compared in 64 bits.  Of equals the
// lowest index comes first.  weights[t, j] = factor * s of the j-th choice, divided by the choices' sum where that is asked for.  Then the (token, choice)
// pairs are put in the experts' order, a token in front of a later one: rows[i] is the token of pair i, places[t, j] is where pair (t, j) went, and
// offsets[e] is where expert e begins: a counting sort, without atomics, so that equal calls give equal bits.
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
    int64_t stride;  // elements between rows of the logits
    int tokens, count, top, dtype, sigmoid, renormalize;
    float factor;
};

template <typename T>
__device__ __forceinline__ T unsigned_max(T a, T b) { return a > b ? a : b; }

template <int CTRL, typename T>
__device__ __forceinline__ T lanes_moved(T x) {
    if constexpr (sizeof(T) == 4) {
        return (T)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
    } else {
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, 0xf, 0xf, true);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CTRL, 0xf, 0xf, true);
        return (uint64_t)hi << 32 | lo;
    }
}

// The largest of the wave's values, the same bits in every lane (rotations within rows of 16 lanes, then the four rows).
template <typename T>
__device__ __forceinline__ T wave_max_of(T x) {
    x = unsigned_max(x, lanes_moved<0x121>(x));
    x = unsigned_max(x, lanes_moved<0x122>(x));
    x = unsigned_max(x, lanes_moved<0x124>(x));
    x = unsigned_max(x, lanes_moved<0x128>(x));
    auto lane = [&](int l) __attribute__((always_inline)) {
        if constexpr (sizeof(T) == 4) return (T)__builtin_amdgcn_readlane((int)x, l);
        else return (T)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), l) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, l));
    };
    return unsigned_max(unsigned_max(lane(0), lane(16)), unsigned_max(lane(32), lane(48)));
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

__device__ __forceinline__ double wave_sum_wide(double v) {
#pragma unroll
    for (int by = 32; by; by >>= 1) v += __shfl_xor(v, by);
    return v;
}

// One wave, one token: expert lane + 64 j in register j.  Choice i's expert (-1: there is none) and weight come back in lane i.
template <int EPL, bool BIAS>
__device__ __forceinline__ void choose_experts(const RouteArgs& a, int experts, int token, int* chosen, float* weight) {
    using Key = std::conditional_t<BIAS, uint64_t, uint32_t>;
    const int lane = threadIdx.x & 63;
    *chosen = -1;
    *weight = 0.f;
    if (a.mask && !a.mask[token]) return;
    float x[EPL], score[EPL];
    Key key[EPL];
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
        const int e = lane + 64 * j;
        const long at = token * a.stride + e;
        x[j] = -INFINITY;
        if (e < experts) {
            if (a.dtype == HFRK_FP32) x[j] = static_cast<const float*>(a.logits)[at];
            else if (a.dtype == HFRK_BF16) x[j] = load16<HFRK_BF16>(static_cast<const uint16_t*>(a.logits)[at]);
            else x[j] = load16<HFRK_F16>(static_cast<const uint16_t*>(a.logits)[at]);
        }
    }
    // scores; the sum over all experts is NaN where a logit is
    float most = x[0], sum = 0.f;
#pragma unroll
    for (int j = 1; j < EPL; ++j) most = fmaxf(most, x[j]);
    most = wave_max(most);
    if (most == -INFINITY) most = 0.f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
        score[j] = a.sigmoid ? 1.0f / (1.0f + expf(-x[j])) : expf(x[j] - most);
        sum += score[j];
    }
    sum = wave_sum(sum);
    if (!a.sigmoid) {
#pragma unroll
        for (int j = 0; j < EPL; ++j) score[j] = score[j] / sum;
    }
    if constexpr (BIAS) {
        double wide[EPL], whole = 0.0;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            wide[j] = a.sigmoid ? 1.0 / (1.0 + exp(-(double)x[j])) : exp((double)x[j] - (double)most);
            whole += wide[j];
        }
        if (!a.sigmoid) whole = wave_sum_wide(whole);
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            const int e = lane + 64 * j;
            const double s = a.sigmoid ? wide[j] : wide[j] / whole;
            key[j] = x[j] > -INFINITY ? order_of(s + (double)(e < experts ? a.bias[e] : 0.f)) : 0;
        }
    } else {
#pragma unroll
        for (int j = 0; j < EPL; ++j) key[j] = order_of(x[j]);
    }

    for (int i = 0; i < a.top; ++i) {
        Key mine = key[0];
#pragma unroll
        for (int j = 1; j < EPL; ++j) mine = unsigned_max(mine, key[j]);
        const Key best = wave_max_of(mine);
        if (best == 0) break;
        bool found = false;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            const uint64_t equal = found ? 0 : __ballot(key[j] == best);
            if (equal) {
                const int owner = __builtin_ctzll(equal);
                const float s = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(score[j]), owner));
                if (lane == owner) key[j] = 0;
                if (lane == i) {
                    *chosen = owner + 64 * j;
                    *weight = s;
                }
                found = true;
            }
        }
    }
    if (a.renormalize) {
        const float part = wave_sum(*weight);
        if (part != 0.f) *weight = *weight / part;
    }
    *weight *= a.factor;
    if (sum != sum) *weight = NAN;
}

// A token a wave; pairs that are nothing get their place here.
template <int EPL, bool BIAS>
__global__ void __launch_bounds__(256) choose_experts_kernel(const RouteArgs a, int experts) {
    const int lane = threadIdx.x & 63, token = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (token >= a.tokens) return;
    int chosen;
    float weight;
    choose_experts<EPL, BIAS>(a, experts, token, &chosen, &weight);
    if (lane < a.top) {
        const long at = (long)token * a.top + lane;
        a.weights[at] = weight;
        a.experts[at] = chosen;
        if (chosen < 0) a.places[at] = -1;
    }
}

// Workgroup e puts expert e's pairs in order: it counts the pairs of lower experts and its own, a wave each sixteenth of them, and then goes through
// its part again.  The last workgroup has what is behind the last expert.
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;

__global__ void __launch_bounds__(kSortThreads) sort_pairs_kernel(const RouteArgs a, int experts) {
    __shared__ int lower[kSortWaves], same[kSortWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), mine = blockIdx.x;
    const int part = ((a.count + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
    const int from = min(wave * part, a.count), to = min(from + part, a.count);
    int below = 0, equal = 0;
#pragma unroll 8
    for (int i = from + lane; i < to; i += 64) {
        const int e = a.experts[i];
        below += (uint32_t)e < (uint32_t)mine;
        equal += e == mine;
    }
    below = __builtin_amdgcn_readlane(wave_prefix_sum(below), 63);
    equal = __builtin_amdgcn_readlane(wave_prefix_sum(equal), 63);
    if (lane == 0) {
        lower[wave] = below;
        same[wave] = equal;
    }
    __syncthreads();
    int start = 0, at = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
        start += lower[w];
        at += w < wave ? same[w] : 0;
    }
    at += start;
    if (threadIdx.x == 0) a.offsets[mine] = start;
    if (mine == experts) {
        for (int i = start + (int)threadIdx.x; i < a.count; i += kSortThreads) a.rows[i] = -1;
        return;
    }
    if (equal == 0) return;
    for (int i = from; i < to; i += 64) {
        const bool hit = i + lane < to && a.experts[i + lane] == mine;
        const uint64_t hits = __ballot(hit);
        if (hit) {
            const int place = at + __builtin_amdgcn_mbcnt_hi((uint32_t)(hits >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hits, 0));
            a.places[i + lane] = place;
            a.rows[place] = (i + lane) / a.top;
        }
        at += __builtin_popcountll(hits);
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

template <int EPL, bool BIAS>
static int launch_route(const RouteArgs& a, int experts, hipStream_t stream) {
    if (a.count <= kFewPairs && a.tokens <= 4 * kSortWaves) {
        hipLaunchKernelGGL((route_few_kernel<EPL, BIAS>), dim3(1), dim3(kSortThreads), 0, stream, a, experts);
    } else {
        hipLaunchKernelGGL((choose_experts_kernel<EPL, BIAS>), dim3((a.tokens + 3) / 4), dim3(256), 0, stream, a, experts);
        HFRK_HIP_TRY(hipGetLastError());
        hipLaunchKernelGGL(sort_pairs_kernel, dim3(experts + 1), dim3(kSortThreads), 0, stream, a, experts);
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

int hfrk_route_experts(const hfrk_route_args* args, void* stream) {
    using namespace hfrk;
    if (!args) return HFRK_BAD_SHAPE;
    RouteArgs a{args->logits, args->bias, static_cast<const uint8_t*>(args->mask), args->weights, args->experts, args->places, args->rows, args->offsets,
                args->logits_stride, args->tokens, 0, args->top, args->dtype, args->sigmoid, args->renormalize, args->factor};
    const int experts = args->num_experts;
    if (a.tokens < 0 || experts < 1 || experts > kMaxExperts || a.top < 1 || a.top > HFRK_MAX_TOP || a.top > experts) return HFRK_BAD_SHAPE;
    if (a.tokens > (1 << 24) || (long)a.tokens * a.top > (1L << 28) || a.stride < 0) return HFRK_BAD_SHAPE;
    if (a.dtype != HFRK_F16 && a.dtype != HFRK_BF16 && a.dtype != HFRK_FP32) return HFRK_BAD_DTYPE;
    if (!a.offsets || (a.tokens && (!a.logits || !a.weights || !a.experts || !a.places || !a.rows))) return HFRK_BAD_SHAPE;
    if ((reinterpret_cast<uintptr_t>(a.bias) | reinterpret_cast<uintptr_t>(a.weights) | reinterpret_cast<uintptr_t>(a.experts) |
         reinterpret_cast<uintptr_t>(a.places) | reinterpret_cast<uintptr_t>(a.rows) | reinterpret_cast<uintptr_t>(a.offsets)) & 3 ||
        reinterpret_cast<uintptr_t>(a.logits) & (a.dtype == HFRK_FP32 ? 3 : 1))
        return HFRK_BAD_ALIGNMENT;
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
