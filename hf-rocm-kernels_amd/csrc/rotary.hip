// Rotary positions, and the append of a step's keys and values to a paged cache with the rotation on the way.
//
//   a_j = position * frequency_j;  pair (x, y) -> magnitude * (x cos a_j - y sin a_j,  y cos a_j + x sin a_j)
//   pairs of a head's first `rotated` values: (j, j + rotated/2), or (2j, 2j+1) interleaved; the values behind them are copied
//
// One workgroup has one token's heads (or a part of them, where there are few tokens): first one thread per pair makes the token's cosine
// and sine and leaves them in LDS, then every thread turns 16 values of a head (two 16-byte pieces) at a time.  Bytes are the bound: 4 a
// value, against 3 multiply-adds; made per value instead of per token the cosines would cost as much as the copy.  The first
// pieces are requested in front of the cosines.
//
// The angle in 32 bits is off by 2^-24 of itself, 0.008 at position 131072: more than bf16's rounding of the result.  Position and frequency are
// multiplied in double, in turns; what is left of the turn fits a float, and an eighth of a turn either way is a short series.
#include "hfrk_internal.h"
#include "overlap.h"

namespace hfrk {

constexpr int kRotaryThreads = 256;

// cos and sin of 2 pi t, t = position * frequency / 2 pi mod 1.  The quadrant is exact; the series end where the next term is below 2^-25 for
// |x| <= pi/4: x^11/11! = 2e-9, x^10/10! = 2.5e-8.  Absolute error below 2^-22: of t as a float 2 pi 2^-26, of x, x^2 and the series' sums the rest.
__device__ __forceinline__ float2 turn(double position, double frequency, float magnitude) {
    const double turns = position * (frequency * 0.15915494309189535);
    const float t = (float)(turns - rint(turns));
    const float quadrant = rintf(4.f * t);
    const float x = fmaf(quadrant, -0.25f, t) * 6.2831853071795865f, z = x * x;
    const float s = fmaf(x * z, fmaf(z, fmaf(z, fmaf(z, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), x);
    const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, 1.f / 40320, -1.f / 720), 1.f / 24), -0.5f), 1.f);
    const int n = (int)quadrant;
    const float cosine = n & 1 ? s : c, sine = n & 1 ? c : s;
    return make_float2((n + 1) & 2 ? -magnitude * cosine : magnitude * cosine, n & 2 ? -magnitude * sine : magnitude * sine);
}

__device__ __forceinline__ long index_at(const void* p, int wide, int i) {
    return wide ? (long)static_cast<const int64_t*>(p)[i] : (long)static_cast<const int32_t*>(p)[i];
}

__device__ __forceinline__ double frequency_at(const void* p, int wide, int i) {
    return wide ? static_cast<const double*>(p)[i] : (double)static_cast<const float*>(p)[i];
}

__device__ __forceinline__ void token_turns(const hfrk_append_args& a, long position, float* cosine, float* sine, int thread, int threads) {
    for (int j = thread; j < a.rotated / 2; j += threads) {
        const float2 cs = turn((double)position, frequency_at(a.frequencies, a.frequencies_wide, j), a.magnitude);
        cosine[j] = cs.x;
        sine[j] = cs.y;
    }
}

// Where a slot's values lie: its page's first element and its place in the page; false for a slot outside the cache (padding).
__device__ __forceinline__ bool slot_place(const hfrk_append_args& a, int token, long& page, long& place) {
    const long slot = index_at(a.slots, a.slots_wide, token);
    if (slot < 0 || slot >= (long)a.pages * a.page_size) return false;
    page = slot < (1L << 31) ? (long)((uint32_t)slot / (uint32_t)a.page_size) : slot / a.page_size;
    place = slot - page * a.page_size;
    return true;
}

template <int DT>
__device__ __forceinline__ void unpack8(uint4 p, float (&x)[8]) {
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        x[2 * j] = load16<DT>((uint16_t)(w[j] & 0xffff));
        x[2 * j + 1] = load16<DT>((uint16_t)(w[j] >> 16));
    }
}

template <int DT>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = (uint32_t)store16<DT>(x[2 * j]) | ((uint32_t)store16<DT>(x[2 * j + 1]) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint2 pack8_fp8(const float (&x)[8], float inv_scale) {
    uint32_t w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        w[j] = cvt_pk_fp8_or_nan(x[4 * j] * inv_scale, x[4 * j + 1] * inv_scale, 0u, false);
        w[j] = cvt_pk_fp8_or_nan(x[4 * j + 2] * inv_scale, x[4 * j + 3] * inv_scale, w[j], true);
    }
    return make_uint2(w[0], w[1]);
}

// One thread's 16 values of one head: what they are and where they go.
struct Pieces {
    const uint16_t* from;  // nullptr: nothing to do
    void* to;
    int first, second;     // offsets of the two pieces in the head
    int pair;              // first of their 8 pairs, or -1: copied
    float inv_scale;
    bool fp8;
};

// Vectorised: a head is head_dim/16 units of 16 values, threadIdx.x the unit, threadIdx.y the head.  Needs 16-byte aligned heads, head_dim and
// rotated multiples of 16.
template <int DT, bool FP8>
__global__ void __launch_bounds__(kRotaryThreads) append_kernel(const hfrk_append_args a) {
    extern __shared__ float turns[];
    float *const cosine = turns, *const sine = turns + a.rotated / 2;
    const int token = blockIdx.x, unit = threadIdx.x;
    const int heads = a.heads + 2 * a.kv_heads, step = blockDim.y * gridDim.y;
    const long position = a.rotated ? index_at(a.positions, a.positions_wide, token) : 0;
    long page = 0, place = 0;
    const bool kept = a.kv_heads > 0 && slot_place(a, token, page, place);
    const int turned = a.rotated / 16;

    auto pieces = [&](int head) {
        Pieces p = {nullptr, nullptr, 0, 0, -1, 1.f, false};
        if (head >= heads) return p;
        if (head < a.heads) {
            p.from = static_cast<const uint16_t*>(a.query) + token * a.query_token_stride + head * a.query_head_stride;
            p.to = static_cast<uint16_t*>(a.query_output) + token * a.output_token_stride + head * a.output_head_stride;
        } else {
            if (!kept) return p;
            const bool value = head >= a.heads + a.kv_heads;
            const int h = head - a.heads - (value ? a.kv_heads : 0);
            p.from = value ? static_cast<const uint16_t*>(a.value) + token * a.value_token_stride + h * a.value_head_stride
                           : static_cast<const uint16_t*>(a.key) + token * a.key_token_stride + h * a.key_head_stride;
            const long at = value ? page * a.value_page_stride + place * a.value_place_stride + h * a.value_cache_head_stride
                                  : page * a.key_page_stride + place * a.key_place_stride + h * a.key_cache_head_stride;
            void* const cache = value ? a.value_cache : a.key_cache;
            if (FP8) {
                p.to = static_cast<uint8_t*>(cache) + at;
                p.fp8 = true;
                const float* const scale = value ? a.value_scale : a.key_scale;
                if (scale) p.inv_scale = 1.f / scale[h * (value ? a.value_scale_stride : a.key_scale_stride)];
            } else {
                p.to = static_cast<uint16_t*>(cache) + at;
            }
            if (value) {
                p.first = 16 * unit;
                p.second = p.first + 8;
                return p;
            }
        }
        if (unit < turned) {
            p.pair = 8 * unit;
            p.first = a.interleaved ? 16 * unit : 8 * unit;
            p.second = a.interleaved ? p.first + 8 : p.first + a.rotated / 2;
        } else {
            p.first = 16 * unit;
            p.second = p.first + 8;
        }
        return p;
    };
    auto load = [&](const Pieces& p, uint4& x, uint4& y) {
        if (!p.from) return;
        x = *reinterpret_cast<const uint4*>(p.from + p.first);
        y = *reinterpret_cast<const uint4*>(p.from + p.second);
    };

    int head = threadIdx.y + blockDim.y * blockIdx.y;
    Pieces p = pieces(head);
    uint4 x = {}, y = {};
    load(p, x, y);
    if (a.rotated) token_turns(a, position, cosine, sine, threadIdx.y * blockDim.x + unit, blockDim.x * blockDim.y);
    __syncthreads();
    while (head < heads) {
        head += step;
        const Pieces next = pieces(head);
        uint4 next_x = {}, next_y = {};
        load(next, next_x, next_y);
        if (p.from) {
            float u[8], v[8];
            unpack8<DT>(x, u);
            unpack8<DT>(y, v);
            if (p.pair >= 0) {
                float c[8], s[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    c[j] = cosine[p.pair + j];
                    s[j] = sine[p.pair + j];
                }
                if (a.interleaved) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float u0 = u[2 * j], u1 = u[2 * j + 1], v0 = v[2 * j], v1 = v[2 * j + 1];
                        u[2 * j] = u0 * c[j] - u1 * s[j];
                        u[2 * j + 1] = u1 * c[j] + u0 * s[j];
                        v[2 * j] = v0 * c[4 + j] - v1 * s[4 + j];
                        v[2 * j + 1] = v1 * c[4 + j] + v0 * s[4 + j];
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float u0 = u[j], v0 = v[j];
                        u[j] = u0 * c[j] - v0 * s[j];
                        v[j] = v0 * c[j] + u0 * s[j];
                    }
                }
            }
            if (FP8 && p.fp8) {
                uint8_t* const to = static_cast<uint8_t*>(p.to);
                *reinterpret_cast<uint2*>(to + p.first) = pack8_fp8(u, p.inv_scale);
                *reinterpret_cast<uint2*>(to + p.second) = pack8_fp8(v, p.inv_scale);
            } else {
                uint16_t* const to = static_cast<uint16_t*>(p.to);
                *reinterpret_cast<uint4*>(to + p.first) = p.pair >= 0 ? pack8<DT>(u) : x;  // (copied values keep their bits, a NaN's too)
                *reinterpret_cast<uint4*>(to + p.second) = p.pair >= 0 ? pack8<DT>(v) : y;
            }
        }
        p = next;
        x = next_x;
        y = next_y;
    }
}

// One pair, or one copied value, a thread and step; any strides, alignment and even `rotated`.
template <int DT, bool FP8>
__global__ void __launch_bounds__(kRotaryThreads) append_scalar_kernel(const hfrk_append_args a) {
    extern __shared__ float turns[];
    float *const cosine = turns, *const sine = turns + a.rotated / 2;
    const int token = blockIdx.x, half = a.rotated / 2, items = a.head_dim - half;
    const long position = a.rotated ? index_at(a.positions, a.positions_wide, token) : 0;
    long page = 0, place = 0;
    const bool kept = a.kv_heads > 0 && slot_place(a, token, page, place);
    if (a.rotated) token_turns(a, position, cosine, sine, threadIdx.x, blockDim.x);
    __syncthreads();

    auto put = [&](void* to, int at, float x, float inv_scale, bool fp8) {
        if (FP8 && fp8) static_cast<uint8_t*>(to)[at] = cvt_fp8_or_nan(x * inv_scale);
        else static_cast<uint16_t*>(to)[at] = store16<DT>(x);
    };
    auto rows = [&](const uint16_t* from, void* to, float inv_scale, bool fp8, int i) {
        if (i < half) {
            const int j = a.interleaved ? 2 * i : i, k = a.interleaved ? j + 1 : i + half;
            const float u = load16<DT>(from[j]), v = load16<DT>(from[k]);
            put(to, j, u * cosine[i] - v * sine[i], inv_scale, fp8);
            put(to, k, v * cosine[i] + u * sine[i], inv_scale, fp8);
        } else if (FP8 && fp8) {
            put(to, i + half, load16<DT>(from[i + half]), inv_scale, fp8);
        } else {
            static_cast<uint16_t*>(to)[i + half] = from[i + half];
        }
    };
    for (int n = threadIdx.x + blockDim.x * blockIdx.y; n < a.heads * items; n += blockDim.x * gridDim.y) {
        const int h = n / items;
        rows(static_cast<const uint16_t*>(a.query) + token * a.query_token_stride + h * a.query_head_stride,
             static_cast<uint16_t*>(a.query_output) + token * a.output_token_stride + h * a.output_head_stride, 1.f, false, n - h * items);
    }
    if (!kept) return;
    constexpr int kSize = FP8 ? 1 : 2;
    for (int n = threadIdx.x + blockDim.x * blockIdx.y; n < a.kv_heads * items; n += blockDim.x * gridDim.y) {
        const int h = n / items;
        const long at = page * a.key_page_stride + place * a.key_place_stride + h * a.key_cache_head_stride;
        rows(static_cast<const uint16_t*>(a.key) + token * a.key_token_stride + h * a.key_head_stride, static_cast<uint8_t*>(a.key_cache) + at * kSize,
             FP8 && a.key_scale ? 1.f / a.key_scale[h * a.key_scale_stride] : 1.f, FP8, n - h * items);
    }
    for (int n = threadIdx.x + blockDim.x * blockIdx.y; n < a.kv_heads * a.head_dim; n += blockDim.x * gridDim.y) {
        const int h = n / a.head_dim, i = n - h * a.head_dim;
        const long at = page * a.value_page_stride + place * a.value_place_stride + h * a.value_cache_head_stride;
        const uint16_t x = static_cast<const uint16_t*>(a.value)[token * a.value_token_stride + h * a.value_head_stride + i];
        if (FP8) static_cast<uint8_t*>(a.value_cache)[at + i] = cvt_fp8_or_nan(load16<DT>(x) * (a.value_scale ? 1.f / a.value_scale[h * a.value_scale_stride] : 1.f));
        else static_cast<uint16_t*>(a.value_cache)[at + i] = x;
    }
}

static bool pieces_of_16(const hfrk_append_args& a, bool fp8) {
    uintptr_t addresses = 0;
    int64_t strides = 0;
    if (a.heads) {
        addresses |= reinterpret_cast<uintptr_t>(a.query) | reinterpret_cast<uintptr_t>(a.query_output);
        strides |= a.query_token_stride | a.query_head_stride | a.output_token_stride | a.output_head_stride;
    }
    if (a.kv_heads) {
        addresses |= reinterpret_cast<uintptr_t>(a.key) | reinterpret_cast<uintptr_t>(a.value);
        const uintptr_t caches = reinterpret_cast<uintptr_t>(a.key_cache) | reinterpret_cast<uintptr_t>(a.value_cache);
        addresses |= fp8 ? caches << 1 : caches;  // 8 values are 8 bytes there
        strides |= a.key_token_stride | a.key_head_stride | a.value_token_stride | a.value_head_stride | a.key_page_stride | a.key_place_stride |
                   a.key_cache_head_stride | a.value_page_stride | a.value_place_stride | a.value_cache_head_stride;
    }
    return a.head_dim % 16 == 0 && a.rotated % 16 == 0 && (addresses & 15) == 0 && (strides & 7) == 0;
}

// The same from token `first` on.
static hfrk_append_args behind(hfrk_append_args a, int64_t first, int tokens) {
    auto ahead = [](const void* p, int64_t bytes) { return p ? static_cast<const uint8_t*>(p) + bytes : nullptr; };
    a.query = ahead(a.query, 2 * first * a.query_token_stride);
    a.query_output = const_cast<uint8_t*>(ahead(a.query_output, 2 * first * a.output_token_stride));
    a.key = ahead(a.key, 2 * first * a.key_token_stride);
    a.value = ahead(a.value, 2 * first * a.value_token_stride);
    a.slots = ahead(a.slots, (a.slots_wide ? 8 : 4) * first);
    a.positions = ahead(a.positions, (a.positions_wide ? 8 : 4) * first);
    a.tokens = tokens;
    return a;
}

// A launch's threads are counted in 32 bits, and one of 2^24 + n workgroups of 256 runs n of them, without an error.
constexpr int kTokensOfALaunch = 1 << 23;

template <int DT, bool FP8>
static int launch_append(const hfrk_append_args& a, hipStream_t stream) {
    if (a.tokens > kTokensOfALaunch) {
        for (int first = 0; first < a.tokens;) {
            const int tokens = a.tokens - first < kTokensOfALaunch ? a.tokens - first : kTokensOfALaunch;
            const int status = launch_append<DT, FP8>(behind(a, first, tokens), stream);
            if (status != HFRK_SUCCESS) return status;
            first += tokens;
        }
        return HFRK_SUCCESS;
    }
    const size_t lds = (size_t)a.rotated * sizeof(float);
    const int heads = a.heads + 2 * a.kv_heads;
    if (pieces_of_16(a, FP8)) {
        const int units = a.head_dim / 16;
        int side = kRotaryThreads / units;
        if (side > heads) side = heads;
        // Few tokens: every thread has one head's piece, and the heads' workgroups make the token's cosines again; from one workgroup per compute
        // unit on the cosines are made once a token.
        const int parts = a.tokens < kNumCU ? (heads + side - 1) / side : 1;
        hipLaunchKernelGGL((append_kernel<DT, FP8>), dim3(a.tokens, parts), dim3(units, side), lds, stream, a);
    } else {
        const int parts = a.tokens < kNumCU ? (int)(((long)heads * a.head_dim + kRotaryThreads - 1) / kRotaryThreads) : 1;
        hipLaunchKernelGGL((append_scalar_kernel<DT, FP8>), dim3(a.tokens, parts < 64 ? parts : 64), dim3(kRotaryThreads), lds, stream, a);
    }
    HFRK_HIP_TRY(hipGetLastError());
    return HFRK_SUCCESS;
}

}  // namespace hfrk

extern "C" int hfrk_append_kv(const hfrk_append_args* args, void* stream) {
    using namespace hfrk;
    if (!args) return HFRK_BAD_SHAPE;
    const hfrk_append_args& a = *args;
    if (a.tokens < 0 || a.heads < 0 || a.kv_heads < 0 || a.heads > 65536 || a.kv_heads > 65536 || a.head_dim < 1 || a.head_dim > 1024) return HFRK_BAD_SHAPE;
    if (a.rotated < 0 || a.rotated > a.head_dim || a.rotated % 2 != 0) return HFRK_BAD_SHAPE;
    if (a.dtype != HFRK_F16 && a.dtype != HFRK_BF16) return HFRK_BAD_DTYPE;
    const bool fp8 = a.kv_heads > 0 && a.cache_dtype == HFRK_FP8_E4M3FN;
    if (a.kv_heads > 0 && !fp8 && a.cache_dtype != a.dtype) return HFRK_BAD_DTYPE;
    if (a.tokens == 0 || a.heads + a.kv_heads == 0) return HFRK_SUCCESS;
    if (a.rotated > 0 && (!a.positions || !a.frequencies)) return HFRK_BAD_SHAPE;
    if (a.heads > 0 && (!a.query || !a.query_output)) return HFRK_BAD_SHAPE;
    if (a.kv_heads > 0) {
        if (!a.key || !a.value || !a.key_cache || !a.value_cache || !a.slots || a.pages < 0 || a.page_size < 1) return HFRK_BAD_SHAPE;
        if (!fp8 && (a.key_scale || a.value_scale)) return HFRK_BAD_DTYPE;
    }
    if (append_overlap(a)) return HFRK_BAD_SHAPE;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (a.dtype == HFRK_F16) return fp8 ? launch_append<HFRK_F16, true>(a, s) : launch_append<HFRK_F16, false>(a, s);
    return fp8 ? launch_append<HFRK_BF16, true>(a, s) : launch_append<HFRK_BF16, false>(a, s);
}

extern "C" int hfrk_rotary(const void* x, int64_t x_token_stride, int64_t x_head_stride, void* output, int64_t output_token_stride,
                           int64_t output_head_stride, const void* positions, int positions_wide, const void* frequencies, int frequencies_wide,
                           float magnitude, int interleaved, int tokens, int heads, int head_dim, int rotated, int dtype, void* stream) {
    hfrk_append_args a = {};
    a.query = x;
    a.query_token_stride = x_token_stride;
    a.query_head_stride = x_head_stride;
    a.query_output = output;
    a.output_token_stride = output_token_stride;
    a.output_head_stride = output_head_stride;
    a.positions = positions;
    a.positions_wide = positions_wide;
    a.frequencies = frequencies;
    a.frequencies_wide = frequencies_wide;
    a.magnitude = magnitude;
    a.interleaved = interleaved;
    a.tokens = tokens;
    a.heads = heads;
    a.head_dim = head_dim;
    a.rotated = rotated;
    a.dtype = dtype;
    return hfrk_append_kv(&a, stream);
}
