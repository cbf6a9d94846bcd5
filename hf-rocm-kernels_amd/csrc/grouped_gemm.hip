// Products of rows grouped by expert (and of one group, in 8-bit integers): the kernel for few rows a group, and the host side.
//   D[i, n] = (base ? base[i, n] : 0) + sa[r_i] * sb[e, n] * sum_k A[r_i, k] * W[e, n, k]      offsets[e] <= i < offsets[e+1], r_i = rows[i] or i
// codes of float8_e4m3fn (sums in fp32) or int8 (sums in int32: exact up to k = 131071, then one conversion), scales applied to the whole sum, one
// rounding to 16 bits.  No counterpart in the reference, whose GEMM has one fp8 weight.
//
// grouped_rows_kernel: a workgroup takes 16 MT rows of a group by 16 RT columns, and its eight waves take the 128-byte chunks of k in turn, so that at
// any time the workgroup reads a run of 1 KB of each weight row.  Operands go from memory to registers (lane l of a 16 x 16 tile holds pieces l / 16 and
// l / 16 + 4 of row l % 16: which bytes of k a lane has does not matter as long as both operands agree); the waves' sums meet in LDS, in wave order.
#include <limits.h>

#include "grouped_gemm.h"

namespace hfrk {

constexpr int kRowsWaves = 8;
constexpr int kRowsChunk = 128;  // bytes of k that a wave takes at a time

template <int DT>
__device__ __forceinline__ uint32_t two_to_16bit(float lo, float hi) {
    return (uint32_t)store16<DT>(lo) | (uint32_t)store16<DT>(hi) << 16;
}

template <bool INT8, int MT, int RT>
__global__ void __launch_bounds__(64 * kRowsWaves) grouped_rows_kernel(const GroupedArgs a) {
    constexpr int U = MT * RT >= 4 ? 2 : 4;  // chunks requested together
    static_assert(MT * RT <= kRowsWaves, "the epilogue has a thread for every four values");
    __shared__ v4i sums[kRowsWaves][MT * RT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    GroupTile t;
    if (!find_tile(a, 16 * MT, &t)) return;
    const int m0 = t.tile % t.tiles_m * 16 * MT, n0 = t.tile / t.tiles_m * 16 * RT;
    const int row0 = t.first + m0, rows = min(16 * MT, t.rows - m0), cols = min(16 * RT, a.n - n0);

    // which row of A a row of the tile is; rows that are none read as zero
    auto row_of_a = [&](int r) __attribute__((always_inline)) {
        const int i = r < rows ? (a.rows ? a.rows[row0 + r] : row0 + r) : -1;
        return (uint32_t)i < (uint32_t)a.a_rows ? i : -1;
    };
    // gathered rows lie anywhere in A (below 2 GB); others behind the tile's first
    const long a_from = a.rows ? 0 : row0;
    const __amdgpu_buffer_rsrc_t ra = make_rsrc(a.A + a_from * a.k, (uint32_t)((a.rows ? a.a_rows : rows) * (long)a.k));
    const __amdgpu_buffer_rsrc_t rb =
        make_rsrc(a.B + t.expert * a.expert_stride + (long)n0 * a.b_stride, (uint32_t)(cols - 1) * (uint32_t)a.b_stride + (uint32_t)a.k);
    const int piece = (lane >> 4) * 16;
    uint32_t va[MT], vb[RT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int r = row_of_a(i * 16 + (lane & 15));
        va[i] = r >= 0 ? (uint32_t)((r - a_from) * a.k + piece) : (uint32_t)kOutsideBuffer;
    }
#pragma unroll
    for (int j = 0; j < RT; ++j) vb[j] = (uint32_t)(j * 16 + (lane & 15)) * (uint32_t)a.b_stride + piece;

    // what the epilogue needs of this thread's four values, requested ahead
    const int e_tile = threadIdx.x >> 6, e_m = e_tile / RT * 16 + (lane & 15), e_n = e_tile % RT * 16 + (lane >> 4) * 4;
    const bool writes = e_tile < MT * RT && e_m < rows && e_n < cols;
    float sa = 0.f, sb[4];
    if (writes) {
        const int r = row_of_a(e_m);
        sa = r >= 0 ? a.scale_a[(long)r * a.sa_stride] : 0.f;
#pragma unroll
        for (int v = 0; v < 4; ++v)
            sb[v] = a.scale_b ? a.scale_b[t.expert * a.sb_expert_stride + (long)min(n0 + e_n + v, a.n - 1) * a.sb_stride] : 1.0f;
    }

    typedef int acc_i __attribute__((ext_vector_type(4)));
    typedef float acc_f __attribute__((ext_vector_type(4)));
    using Acc = std::conditional_t<INT8, acc_i, acc_f>;
    Acc acc[MT][RT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[i][j] = Acc{0, 0, 0, 0};

    const int chunks = (a.k + kRowsChunk - 1) / kRowsChunk;
#pragma unroll 1
    for (int c = wave; c < chunks; c += kRowsWaves * U) {
        v4i fa[U][MT][2], fb[U][RT][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kb = (c + u * kRowsWaves) * kRowsChunk;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bool inside = kb + h * 64 + piece < a.k;
                const uint32_t by = (uint32_t)(kb + h * 64);
#pragma unroll
                for (int j = 0; j < RT; ++j) fb[u][j][h] = __builtin_amdgcn_raw_buffer_load_b128(rb, inside ? vb[j] + by : (uint32_t)kOutsideBuffer, 0, 0);
#pragma unroll
                for (int i = 0; i < MT; ++i) fa[u][i][h] = __builtin_amdgcn_raw_buffer_load_b128(ra, inside ? va[i] + by : (uint32_t)kOutsideBuffer, 0, 0);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    if constexpr (INT8) {
                        acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[u][j][0], fa[u][i][0], acc[i][j], 0, 0, 0);
                        acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[u][j][1], fa[u][i][1], acc[i][j], 0, 0, 0);
                    } else {
                        auto join = [](v4i lo, v4i hi) __attribute__((always_inline)) { return v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}; };
                        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(join(fb[u][j][0], fb[u][j][1]), join(fa[u][i][0], fa[u][i][1]),
                                                                                      acc[i][j], 0, 0, 0, 0, 0, 0);
                    }
                }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < RT; ++j) sums[wave][i * RT + j][lane] = __builtin_bit_cast(v4i, acc[i][j]);
    __syncthreads();
    if (!writes) return;
    Acc total = Acc{0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < kRowsWaves; ++w) total += __builtin_bit_cast(Acc, sums[w][e_tile][lane]);

    const long at = (long)(row0 + e_m) * a.n + n0 + e_n, base_at = (long)(row0 + e_m) * a.base_stride + n0 + e_n;
    uint16_t* const d = static_cast<uint16_t*>(a.D) + at;
    const uint16_t* const base = a.base ? static_cast<const uint16_t*>(a.base) + base_at : nullptr;
    auto finish = [&](auto dt) __attribute__((always_inline)) {
        constexpr int DT = decltype(dt)::value;
        float x[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) x[v] = (float)total[v] * (sa * sb[v]);
        if (a.vec) {
            if (base) {
                const uint2 b = *reinterpret_cast<const uint2*>(base);
                x[0] += load16<DT>((uint16_t)(b.x & 0xffff));
                x[1] += load16<DT>((uint16_t)(b.x >> 16));
                x[2] += load16<DT>((uint16_t)(b.y & 0xffff));
                x[3] += load16<DT>((uint16_t)(b.y >> 16));
            }
            *reinterpret_cast<uint2*>(d) = make_uint2(two_to_16bit<DT>(x[0], x[1]), two_to_16bit<DT>(x[2], x[3]));
        } else {
#pragma unroll
            for (int v = 0; v < 4; ++v)
                if (n0 + e_n + v < a.n) d[v] = store16<DT>(x[v] + (base ? load16<DT>(base[v]) : 0.f));
        }
    };
    if (a.d_dtype == HFRK_BF16) finish(std::integral_constant<int, HFRK_BF16>{});
    else finish(std::integral_constant<int, HFRK_F16>{});
}

template <bool INT8, int MT, int RT>
static int launch_rows(GroupedArgs a, hipStream_t stream) {
    a.tiles_n = (a.n + 16 * RT - 1) / (16 * RT);
    const long tiles = (a.offsets ? grouped_tiles_bound(a.count, a.experts, 16 * MT) : ((long)a.count + 16 * MT - 1) / (16 * MT)) * a.tiles_n;
    if (tiles * 64 * kRowsWaves > (long)UINT_MAX) return HFRK_BAD_SHAPE;
    hipLaunchKernelGGL((grouped_rows_kernel<INT8, MT, RT>), dim3((unsigned)tiles), dim3(64 * kRowsWaves), 0, stream, a);
    HFRK_HIP_TRY(hipGetLastError());
    return HFRK_SUCCESS;
}

template <bool INT8>
static int launch_grouped(const GroupedArgs& a, hipStream_t stream) {
    return launch_rows<INT8, 1, 2>(a, stream);
}

static int grouped_run(GroupedArgs& a, int type, hipStream_t stream) {
    // offsets inside a tile's buffers stay below 2^31, and the largest int8 product, 2^14 k, below it too
    constexpr int kMost = 1 << 21;
    if (a.count < 0 || a.a_rows < 0 || a.experts < 1 || a.experts > kMaxExperts || a.n < 1 || a.n > kMost || a.k < 1 || a.k > kMost) return HFRK_BAD_SHAPE;
    if (type != HFRK_FP8_E4M3FN && type != HFRK_INT8) return HFRK_BAD_DTYPE;
    if (a.d_dtype != HFRK_F16 && a.d_dtype != HFRK_BF16) return HFRK_BAD_DTYPE;
    if (a.k % 16 != 0) return HFRK_K_NOT_DIVISIBLE_BY_WARPTILE_K;
    if (type == HFRK_INT8 && a.k > 131056) return HFRK_BAD_SHAPE;
    if (a.count == 0) return HFRK_SUCCESS;
    if (!a.A || !a.B || !a.D || !a.scale_a) return HFRK_BAD_SHAPE;
    if (a.b_stride < a.k || a.b_stride > kMost || a.expert_stride < 0) return HFRK_BAD_SHAPE;
    if ((a.sa_stride != 0 && a.sa_stride != 1) || (a.sb_stride != 0 && a.sb_stride != 1) || a.sb_expert_stride < 0) return HFRK_BAD_SHAPE;
    if (a.base && a.base_stride != 0 && (a.base_stride < a.n || a.base_stride > kMost)) return HFRK_BAD_SHAPE;
    if (a.rows ? (long)a.a_rows * a.k > kOutsideBuffer - kMost : a.a_rows < a.count) return HFRK_BAD_SHAPE;
    if ((reinterpret_cast<uintptr_t>(a.A) | reinterpret_cast<uintptr_t>(a.B)) & 15 || (a.b_stride & 15) || (a.expert_stride & 15)) return HFRK_BAD_ALIGNMENT;
    if ((reinterpret_cast<uintptr_t>(a.D) | reinterpret_cast<uintptr_t>(a.base)) & 1) return HFRK_BAD_ALIGNMENT;
    if ((reinterpret_cast<uintptr_t>(a.rows) | reinterpret_cast<uintptr_t>(a.offsets) | reinterpret_cast<uintptr_t>(a.scale_a) |
         reinterpret_cast<uintptr_t>(a.scale_b)) & 3)
        return HFRK_BAD_ALIGNMENT;
    if (!a.base) a.base_stride = 0;
    a.vec = a.n % 4 == 0 && a.base_stride % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.D) | reinterpret_cast<uintptr_t>(a.base)) & 7) == 0;
    return type == HFRK_INT8 ? launch_grouped<true>(a, stream) : launch_grouped<false>(a, stream);
}

}  // namespace hfrk

extern "C" {

int hfrk_grouped_gemm(const hfrk_grouped_args* args, void* stream) {
    if (!args || (!args->offsets && args->count > 0)) return HFRK_BAD_SHAPE;
    hfrk::GroupedArgs a{};
    a.A = static_cast<const uint8_t*>(args->a);
    a.B = static_cast<const uint8_t*>(args->b);
    a.D = args->output;
    a.scale_a = args->scale_a;
    a.scale_b = args->scale_b;
    a.offsets = args->offsets;
    a.rows = args->rows;
    a.expert_stride = args->expert_stride;
    a.sb_expert_stride = args->scale_b ? args->scale_b_expert_stride : 0;
    a.b_stride = args->b_stride;
    a.sa_stride = args->scale_a_stride;
    a.sb_stride = args->scale_b_stride;
    a.count = args->count;
    a.a_rows = args->a_rows;
    a.experts = args->experts;
    a.n = args->n;
    a.k = args->k;
    a.d_dtype = args->dtype;
    return hfrk::grouped_run(a, args->type, static_cast<hipStream_t>(stream));
}

int hfrk_int8_gemm(const void* A, const void* B, void* D, const void* base, int base_stride, const float* scale_a, int sa_stride, const float* scale_b,
                   int sb_stride, int m, int n, int k, int b_stride, int d_dtype, void* stream) {
    hfrk::GroupedArgs a{};
    a.A = static_cast<const uint8_t*>(A);
    a.B = static_cast<const uint8_t*>(B);
    a.D = D;
    a.base = base;
    a.base_stride = base_stride;
    a.scale_a = scale_a;
    a.scale_b = scale_b;
    a.b_stride = b_stride;
    a.sa_stride = sa_stride;
    a.sb_stride = scale_b ? sb_stride : 0;
    a.count = a.a_rows = m;
    a.experts = 1;
    a.n = n;
    a.k = k;
    a.d_dtype = d_dtype;
    return hfrk::grouped_run(a, HFRK_INT8, static_cast<hipStream_t>(stream));
}

}  // extern "C"
