// Stands in for the HIP headers when a kernel's source is compiled for the CPU: the names and the gfx950 builtins that the kernels of attention and of the
// append use.  Every lane runs by itself until it meets a builtin that looks at other lanes of its wave, where it waits for them (lanes.cpp).
// Test infrastructure only.
#pragma once

#include <math.h>
#include <stddef.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <functional>

#define __global__
#define __device__
#define __host__
#define __forceinline__ inline
#define __launch_bounds__(...)
#define __shared__ static  // (one workgroup runs at a time)
#define __align__(n) __attribute__((aligned(n)))

using std::max;
using std::min;
inline uint32_t min(uint32_t a, int b) { return min(a, (uint32_t)b); }
inline long max(long a, int b) { return max(a, (long)b); }

struct dim3 {
    unsigned x, y, z;
    dim3(unsigned x = 1, unsigned y = 1, unsigned z = 1) : x(x), y(y), z(z) {}
};
struct float2 { float x, y; };
struct uint2 { unsigned x, y; };
struct uint4 { unsigned x, y, z, w; };
struct int4 { int x, y, z, w; };
inline float2 make_float2(float x, float y) { return {x, y}; }
inline uint2 make_uint2(unsigned x, unsigned y) { return {x, y}; }
inline uint4 make_uint4(unsigned x, unsigned y, unsigned z, unsigned w) { return {x, y, z, w}; }
inline int4 make_int4(int x, int y, int z, int w) { return {x, y, z, w}; }

// ---- host side
typedef void* hipStream_t;
typedef int hipError_t;
enum { hipSuccess = 0 };
inline hipError_t hipGetLastError() { return hipSuccess; }
namespace lanes {
extern dim3 thread, block, threads, blocks;
extern char dynamic_memory[];  // the launch's own LDS
void launch(dim3 blocks, dim3 threads, const std::function<void()>& kernel);
}  // namespace lanes
#define threadIdx lanes::thread
#define blockIdx lanes::block
#define blockDim lanes::threads
#define gridDim lanes::blocks
#define hipLaunchKernelGGL(kernel, grid, block, lds, stream, ...) lanes::launch(grid, block, [&] { (kernel)(__VA_ARGS__); })

// ---- one lane's arithmetic
template <typename TO, typename FROM>
inline TO bits(FROM from) {
    static_assert(sizeof(TO) == sizeof(FROM), "the same number of bits");
    TO to;
    memcpy(&to, &from, sizeof to);
    return to;
}
inline float __uint_as_float(uint32_t u) { return bits<float>(u); }
inline uint32_t __float_as_uint(float f) { return bits<uint32_t>(f); }
inline uint32_t __umulhi(uint32_t a, uint32_t b) { return (uint64_t)a * b >> 32; }
inline int __ffsll(unsigned long long v) { return __builtin_ffsll(v); }

struct __half { _Float16 h; };
inline float __half2float(__half x) { return (float)x.h; }
inline __half __float2half_rn(float x) { return {(_Float16)x}; }
inline __half __ushort_as_half(uint16_t x) { return {bits<_Float16>(x)}; }
inline uint16_t __half_as_ushort(__half x) { return bits<uint16_t>(x.h); }

namespace lanes {
struct Bf16 {
    static float wide(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
    static uint16_t narrow(float f) {  // (of values that the type holds)
        return f != f ? __float_as_uint(f) >> 16 | 0x40 : __float_as_uint(f) >> 16;
    }
};
struct F16 {
    static float wide(uint16_t b) { return (float)bits<_Float16>(b); }
    static uint16_t narrow(float f) { return bits<uint16_t>((_Float16)f); }
};

inline float from_e4m3(uint8_t b) {
    if ((b & 0x7f) == 0x7f) return NAN;
    const int e = b >> 3 & 15, m = b & 7;
    const float v = e ? ldexpf(1 + m / 8.f, e - 7) : ldexpf(m / 8.f, -6);
    return b & 0x80 ? -v : v;
}
inline uint8_t to_e4m3(float f) {  // nearest, ties to even; of NaN and values up to 448
    if (f != f) return signbit(f) ? 0xff : 0x7f;
    uint8_t best = 0;
    for (int code = 1; code < 127; ++code) {
        const float now = fabsf(fabsf(f) - from_e4m3(code)), before = fabsf(fabsf(f) - from_e4m3(best));
        if (now < before || (now == before && code % 2 == 0)) best = code;
    }
    return best | (signbit(f) ? 0x80 : 0);
}
template <typename T>
inline uint32_t widen_pair(int word, float, bool high) {
    const uint32_t pair = high ? (uint32_t)word >> 16 : (uint32_t)word & 0xffff;
    return T::narrow(from_e4m3(pair & 255)) | (uint32_t)T::narrow(from_e4m3(pair >> 8)) << 16;
}
inline uint32_t narrow_pair(float a, float b, uint32_t old, bool high) {
    const uint32_t pair = to_e4m3(a) | (uint32_t)to_e4m3(b) << 8;
    return high ? (old & 0xffff) | pair << 16 : (old & 0xffff0000u) | pair;
}
inline float median(float a, float b, float c) {
    if (a != a) return fminf(b, c);
    return fmaxf(fminf(a, b), fminf(fmaxf(a, b), c));
}
inline uint32_t permute_bytes(uint32_t high, uint32_t low, uint32_t which) {
    const uint64_t all = (uint64_t)high << 32 | low;
    uint32_t r = 0;
    for (int i = 0; i < 4; ++i) r |= (uint32_t)(all >> 8 * (which >> 8 * i & 255) & 255) << 8 * i;
    return r;
}
template <typename T, typename V>
inline float dot2(V a, V b, float c, bool) {
    const uint32_t x = bits<uint32_t>(a), y = bits<uint32_t>(b);
    return c + T::wide(x & 0xffff) * T::wide(y & 0xffff) + T::wide(x >> 16) * T::wide(y >> 16);
}

// ---- across lanes
struct Words { uint32_t w[8]; };
struct Seen {
    const Words* of;    // what each of the wave's lanes gave
    uint64_t arrived;
    int lane;
};
Seen meet_wave(const Words& mine);
void meet_block();

typedef unsigned Pair __attribute__((ext_vector_type(2)));
template <int N>
inline Pair swap_rows(unsigned a, unsigned b, bool, bool) {  // a's odd rows of N lanes change places with b's even ones
    const Seen s = meet_wave({{a, b}});
    const bool odd = s.lane / N & 1;
    return odd ? Pair{s.of[s.lane - N].w[1], s.of[s.lane].w[1]} : Pair{s.of[s.lane].w[0], s.of[s.lane + N].w[0]};
}
template <typename T>
inline T dpp(T old, T v, int control, int row_mask, int, bool zero) {
    const Seen s = meet_wave({{(unsigned)v}});
    const int row = s.lane / 16, i = s.lane % 16;
    if (!(row_mask >> row & 1)) return old;
    int from = -1;
    if (control > 0x110 && control < 0x120) from = i >= control - 0x110 ? s.lane - (control - 0x110) : -1;  // shift right
    else if (control > 0x120 && control < 0x130) from = row * 16 + (i - (control - 0x120) & 15);              // rotate right
    else if (control == 0x142) from = row ? row * 16 - 1 : -1;                                                  // the row in front's last
    else if (control == 0x143) from = s.lane >= 32 ? 31 : -1;                                                   // the first half's last
    else __builtin_trap();
    return from < 0 ? (zero ? (T)0 : old) : (T)s.of[from].w[0];
}
inline int read_lane(int v, int n) { return (int)meet_wave({{(unsigned)v}}).of[n & 63].w[0]; }
inline int read_first_lane(int v) {
    const Seen s = meet_wave({{(unsigned)v}});
    return (int)s.of[__builtin_ctzll(s.arrived)].w[0];
}

// Rows of A and columns of B are lane % ROWS, eight values of k a lane from 8 * (lane / ROWS) on; C: column lane % ROWS, rows in fours.
template <typename T, int ROWS, typename A, typename C>
inline C product(A a, A b, C c, int, int, int) {
    Words mine;
    memcpy(mine.w, &a, 16);
    memcpy(mine.w + 4, &b, 16);
    const Seen s = meet_wave(mine);
    constexpr int kGroups = 64 / ROWS;
    for (int v = 0; v < (int)(sizeof c / sizeof c[0]); ++v) {
        const int row = v / 4 * 4 * kGroups + 4 * (s.lane / ROWS) + v % 4;
        float sum = c[v];
        for (int g = 0; g < kGroups; ++g) {
            uint16_t x[8], y[8];
            memcpy(x, s.of[ROWS * g + row].w, 16);
            memcpy(y, s.of[ROWS * g + s.lane % ROWS].w + 4, 16);
            for (int k = 0; k < 8; ++k) sum += T::wide(x[k]) * T::wide(y[k]);
        }
        c[v] = sum;
    }
    return c;
}
}  // namespace lanes

inline uint64_t __ballot(int p) {
    const lanes::Seen s = lanes::meet_wave({{p != 0}});
    uint64_t r = 0;
    for (int i = 0; i < 64; ++i) r |= (uint64_t)((s.arrived >> i & 1) && s.of[i].w[0]) << i;
    return r;
}
inline int __any(int p) { return __ballot(p) != 0; }
inline float __shfl_xor(float v, int by) {
    const lanes::Seen s = lanes::meet_wave({{__float_as_uint(v)}});
    return __uint_as_float(s.of[s.lane ^ by].w[0]);
}
#define __syncthreads lanes::meet_block

// Resources of bounded loads, which these kernels do not use: declared for the shared header's sake.
namespace lanes {
struct Resource {};
inline uint4 no_load(Resource, int, int, int) { __builtin_trap(); }
template <typename V>
inline void no_store(V, Resource, int, int, int) { __builtin_trap(); }
}  // namespace lanes
#define __amdgpu_buffer_rsrc_t lanes::Resource
#define __builtin_amdgcn_make_buffer_rsrc(...) lanes::Resource()
#define __builtin_amdgcn_raw_buffer_load_b128 lanes::no_load
#define __builtin_amdgcn_raw_buffer_store_b128 lanes::no_store
#define __builtin_amdgcn_raw_buffer_store_b64 lanes::no_store

#define __builtin_amdgcn_exp2f exp2f
#define __builtin_amdgcn_rcpf(x) (1.f / (x))
#define __builtin_amdgcn_fmed3f lanes::median
#define __builtin_amdgcn_perm lanes::permute_bytes
#define __builtin_amdgcn_cvt_pk_fp8_f32 lanes::narrow_pair
#define __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8 lanes::widen_pair<lanes::Bf16>
#define __builtin_amdgcn_cvt_scalef32_pk_f16_fp8 lanes::widen_pair<lanes::F16>
#define __builtin_amdgcn_fdot2_f32_bf16 lanes::dot2<lanes::Bf16>
#define __builtin_amdgcn_fdot2 lanes::dot2<lanes::F16>
#define __builtin_amdgcn_permlane32_swap lanes::swap_rows<32>
#define __builtin_amdgcn_permlane16_swap lanes::swap_rows<16>
#define __builtin_amdgcn_update_dpp lanes::dpp
#define __builtin_amdgcn_readlane lanes::read_lane
#define __builtin_amdgcn_readfirstlane lanes::read_first_lane
#define __builtin_amdgcn_mfma_f32_16x16x32_bf16 lanes::product<lanes::Bf16, 16>
#define __builtin_amdgcn_mfma_f32_16x16x32_f16 lanes::product<lanes::F16, 16>
#define __builtin_amdgcn_mfma_f32_32x32x16_bf16 lanes::product<lanes::Bf16, 32>
#define __builtin_amdgcn_mfma_f32_32x32x16_f16 lanes::product<lanes::F16, 32>
#define __builtin_amdgcn_s_barrier lanes::meet_block
#define __builtin_amdgcn_wave_barrier() lanes::meet_wave({})
#define __builtin_amdgcn_fence(...)
