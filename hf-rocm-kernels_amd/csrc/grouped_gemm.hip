// Products of rows grouped by expert (and of one group, in 8-bit integers): the kernel for few rows a group, and the host side.
//   D[i, n] = (base ? base[i, n] : 0) + sa[r_i] * sb[e, n] * sum_k A[r_i, k] * W[e, n, k]      offsets[e] <= i < offsets[e+1], r_i = rows[i] or i
// codes of float8_e4m3fn (sums as the matrix cores make them: a run of eight products is aligned to its largest and loses what is below 2^-13 of that; runs are
// added in fp32) or int8 (sums in int32: exact up to k = 131071, then one conversion), the two scales' product applied to the whole sum, one
// rounding to 16 bits.  No counterpart in the reference, whose GEMM has one fp8 weight.
//
// grouped_rows_kernel: a workgroup takes 16 rows of a group; each of its waves takes 16 RT columns and every KW-th 128-byte chunk of k, so that KW waves
// read a run of KW * 128 bytes of each weight row at a time.  Operands go from memory to registers (lane l of a 16 x 16 tile holds pieces l / 16 and
// l / 16 + 4 of row l % 16: which bytes of k a lane has does not matter as long as both operands agree), one tile's chunk ahead of the one that is
// multiplied; the sums of the waves along k meet in LDS, in wave order.  Bound by memory: 5.8 TB/s on 940 MB of weights.  More rows a group go to the tiled
// kernel (tiled_gemm_kernel.h).  One int8 weight goes, by rows and k, to the skinny GEMM's kernels, to this one, or to the tiled one (launch_int8).
#include <limits.h>
#include <math.h>

#include "grouped_gemm.h"
#include "skinny_gemm_args.h"
#include "skinny_gemm_plan.h"

namespace hfrk {

constexpr int kRowsChunk = 128;  // bytes of k that a wave takes at a time
constexpr int kRowsTile = 16;    // rows of a workgroup

template <int DT>
__device__ __forceinline__ uint32_t two_to_16bit(float lo, float hi) {
    return (uint32_t)store16<DT>(lo) | (uint32_t)store16<DT>(hi) << 16;
}

// KW waves split k, CW of them the columns.
template <bool INT8, int RT, int KW, int CW>
__global__ void __launch_bounds__(64 * KW * CW, KW * CW > 8 ? 8 : 6) grouped_rows_kernel(const GroupedArgs a) {
    constexpr int WAVES = KW * CW, TILES = CW * RT;        // matrix tiles of 16 x 16 of the workgroup
    constexpr int EACH = (TILES + WAVES - 1) / WAVES;     // tiles whose sums a wave finishes
    constexpr int BM = kRowsTile, BN = 16 * RT * CW;
    __shared__ v4i sums[KW][TILES][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kw = wave % KW, cw = wave / KW;

    GroupTile t;
    if (!find_tile(a, BM, &t)) return;
    const int m0 = t.tile % t.tiles_m * BM, n0 = t.tile / t.tiles_m * BN;
    const int row0 = t.first + m0, rows = min(BM, t.rows - m0), cols = min(BN, a.n - n0);

    // Which row of A a row of the tile is, -1: none.  The numbers come through a buffer over the tile's own, so that none is read behind them.
    const __amdgpu_buffer_rsrc_t rnumbers = make_rsrc(a.rows + row0, a.rows ? (uint32_t)rows * 4u : 0u);
    auto number_of = [&](int r) __attribute__((always_inline)) { return a.rows ? __builtin_amdgcn_raw_buffer_load_b32(rnumbers, r * 4, 0, 0) : row0 + r; };
    auto row_of = [&](int r, int number) __attribute__((always_inline)) { return r < rows && (uint32_t)number < (uint32_t)a.a_rows ? number : -1; };
    const int number = number_of(lane & 15);

    // gathered rows lie anywhere in A (below 2 GB); others behind the tile's first
    const long a_from = a.rows ? 0 : row0;
    const __amdgpu_buffer_rsrc_t ra = make_rsrc(a.A + a_from * a.k, (uint32_t)((a.rows ? a.a_rows : rows) * (long)a.k));
    const __amdgpu_buffer_rsrc_t rb =
        make_rsrc(a.B + t.expert * a.expert_stride + (long)n0 * a.b_stride, (uint32_t)(cols - 1) * (uint32_t)a.b_stride + (uint32_t)a.k);
    const int piece = (lane >> 4) * 16;
    uint32_t va, vb[RT];
#pragma unroll
    for (int j = 0; j < RT; ++j) vb[j] = (uint32_t)((cw * RT + j) * 16 + (lane & 15)) * (uint32_t)a.b_stride + piece;

    typedef float acc_f __attribute__((ext_vector_type(4)));
    using Acc = std::conditional_t<INT8, v4i, acc_f>;
    Acc acc[RT];
#pragma unroll
    for (int j = 0; j < RT; ++j) acc[j] = Acc{0, 0, 0, 0};

    // registers of the tile that is multiplied and of the next one: a tile's own, or with one tile those of every other chunk
    v4i fa[2][2], fb[RT == 1 ? 2 : RT][2];
    auto get_b = [&](int set, int j, int c) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int by = c * kRowsChunk + h * 64;
            fb[RT == 1 ? set : j][h] = __builtin_amdgcn_raw_buffer_load_b128(rb, by + piece < a.k ? vb[j] + (uint32_t)by : (uint32_t)kOutsideBuffer, 0, 0);
        }
    };
    auto get_a = [&](int set, int c) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int by = c * kRowsChunk + h * 64;
            fa[set][h] = __builtin_amdgcn_raw_buffer_load_b128(ra, by + piece < a.k ? va + (uint32_t)by : (uint32_t)kOutsideBuffer, 0, 0);
        }
    };
    auto multiply = [&](int set, int j) __attribute__((always_inline)) {
        const v4i(&b)[2] = fb[RT == 1 ? set : j];
        if constexpr (INT8) {
            acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[0], fa[set][0], acc[j], 0, 0, 0);
            acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[1], fa[set][1], acc[j], 0, 0, 0);
        } else {
            auto join = [](v4i lo, v4i hi) __attribute__((always_inline)) { return v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}; };
            acc[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(join(b[0], b[1]), join(fa[set][0], fa[set][1]), acc[j], 0, 0, 0, 0, 0, 0);
        }
    };

    // The weight is requested in front of the rows, whose numbers are still on their way.
    const int chunks = (a.k + kRowsChunk - 1) / kRowsChunk;
    get_b(0, 0, kw);
    const int mine = row_of(lane & 15, number);
    va = mine >= 0 ? (uint32_t)((mine - a_from) * a.k + piece) : (uint32_t)kOutsideBuffer;
    get_a(0, kw);
    for (int c = kw; c < chunks; c += 2 * KW) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            get_a(half ^ 1, c + (half + 1) * KW);
#pragma unroll
            for (int j = 0; j < RT; ++j) {
                get_b((half + (j + 1) / RT) & 1, (j + 1) % RT, c + (half + (j + 1) / RT) * KW);
                __builtin_amdgcn_sched_barrier(0);
                multiply(half, j);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < RT; ++j) sums[kw][cw * RT + j][lane] = __builtin_bit_cast(v4i, acc[j]);
    // what the epilogue needs of this thread's values: tile e of the workgroup is columns 16 e and on
    const int e_m = lane & 15, from = row_of(e_m, number_of(e_m));
    const float sa = from >= 0 ? a.scale_a[(long)from * a.sa_stride] : 0.f;
    int e_n[EACH];
    float sb[EACH][4];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        e_n[e] = (wave + e * WAVES) * 16 + (lane >> 4) * 4;
#pragma unroll
        for (int v = 0; v < 4; ++v)
            sb[e][v] = a.scale_b ? a.scale_b[t.expert * a.sb_expert_stride + (long)min(n0 + e_n[e] + v, a.n - 1) * a.sb_stride] : 1.0f;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int tile = wave + e * WAVES;
        if (tile >= TILES || e_m >= rows || e_n[e] >= cols) continue;
        Acc total = Acc{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < KW; ++w) total += __builtin_bit_cast(Acc, sums[w][tile][lane]);
        const long at = (long)(row0 + e_m) * a.n + n0 + e_n[e], base_at = (long)(row0 + e_m) * a.base_stride + n0 + e_n[e];
        uint16_t* const d = static_cast<uint16_t*>(a.D) + at;
        const uint16_t* const base = a.base ? static_cast<const uint16_t*>(a.base) + base_at : nullptr;
        auto finish = [&](auto dt) __attribute__((always_inline)) {
            constexpr int DT = decltype(dt)::value;
            float x[4];
#pragma unroll
            for (int v = 0; v < 4; ++v) x[v] = (float)total[v] * (sa * sb[e][v]);
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
                    if (e_n[e] + v < cols) d[v] = store16<DT>(x[v] + (base ? load16<DT>(base[v]) : 0.f));
            }
        };
        if (a.d_dtype == HFRK_BF16) finish(std::integral_constant<int, HFRK_BF16>{});
        else finish(std::integral_constant<int, HFRK_F16>{});
    }
}

template <bool INT8, int RT, int KW, int CW>
static int launch_rows(GroupedArgs a, hipStream_t stream) {
    constexpr int BN = 16 * RT * CW, THREADS = 64 * KW * CW;
    a.tiles_n = (a.n + BN - 1) / BN;
    const long tiles = (a.offsets ? grouped_tiles_bound(a.count, a.experts, kRowsTile) : ((long)a.count + kRowsTile - 1) / kRowsTile) * a.tiles_n;
    if (tiles * THREADS > (long)UINT_MAX) return HFRK_BAD_SHAPE;
    hipLaunchKernelGGL((grouped_rows_kernel<INT8, RT, KW, CW>), dim3((unsigned)tiles), dim3(THREADS), 0, stream, a);
    HFRK_HIP_TRY(hipGetLastError());
    return HFRK_SUCCESS;
}

// Which rows kernel, and its predicted time in us: rounds of workgroups over the compute units, each reading its columns' weights, its rows (with less weight,
// as they come from L2) and spending the time of 10 KB on its start and end, at 22 KB a us.  `active` groups of `rows` rows.  64 columns a workgroup where there
// are many, in four tiles a wave; a wave asks for one tile's chunk at a time, and it is the six waves of a SIMD that keep memory busy: with all four tiles'
// chunks requested together and two sets of registers 100 tokens on 6 of 160 experts of 3008 x 5120 take 471 us instead of 376 (5.9 TB/s), 32 on 2 of 8 of 28672 x
// 4096 177 and 164.  Fewer columns spread a call over the compute units: one token on 2 of 8 experts of 4096 x 14336 28.9 -> 18.8 us with 32 columns (128 and
// 256 workgroups), on 6 of 64 of 2816 x 2048 12.2 -> 10.1 with 48, one row of 4096 x 14336 int8 29.2 -> 12.9 with 16 (such a weight now goes to int8_skinny); where the rounds do not get fewer they cost (32
// tokens on 2 of 8 of 4096 x 14336 85 -> 113 with 16 columns).  Up to eight chunks of k leave eight waves one each: four waves take k then, and the others other
// columns (4 tokens on 8 of 128 of 2048 x 768 15.8 -> 12.0 with 128 columns, one token 7.5 -> 6.5 with 64 of them).
struct FewRows {
    int cols, waves_k;
    float us;
};

static FewRows few_rows_kernel(int n, int k, float active, float rows) {
    auto workgroups = [&](int cols) { return active * ((n + cols - 1) / cols); };
    auto predicted = [&](int cols) { return 1.5f + ceilf(workgroups(cols) / kNumCU) * (cols + .6f * fminf(rows, 16.f) + 1e4f / k) * k / 22e3f; };
    if (k <= 8 * kRowsChunk) {
        const int cols = workgroups(128) >= kNumCU ? 128 : 64;
        return {cols, 4, predicted(cols)};
    }
    FewRows best{64, 8, predicted(64)};
    for (int cols : {48, 32, 16})
        if (predicted(cols) < best.us) best = {cols, 8, predicted(cols)};
    return best;
}

template <bool INT8>
static int launch_few_rows(const GroupedArgs& a, const FewRows& f, hipStream_t stream) {
    if (f.waves_k == 4) return f.cols == 128 ? launch_rows<INT8, 4, 4, 2>(a, stream) : launch_rows<INT8, 2, 4, 2>(a, stream);
    switch (f.cols) {
        case 64: return launch_rows<INT8, 4, 8, 1>(a, stream);
        case 48: return launch_rows<INT8, 3, 8, 1>(a, stream);
        case 32: return launch_rows<INT8, 2, 8, 1>(a, stream);
        default: return launch_rows<INT8, 1, 8, 1>(a, stream);
    }
}

// The tile shape with the smallest predicted time, in us: rounds of workgroups, each a start and end and k's stages, or the weights' way from memory.  Group sizes
// are not known here: groups of the mean size are assumed, of whose rows of tiles half a one more is partly filled.  Constants fitted to 38 sizes (16 to 2048
// rows a group, k 256 to 14336): the choice is 0.8 % slower than the best shape in the mean, 22 % on the worst (512 tokens, 2 of 8, 4096 x 14336 of very uneven
// popularity: whether a group passes 256 rows decides there).
static int grouped_shape(const GroupedArgs& a, int groups) {
    struct Shape { float fixed, stage, pair_fixed, pair_stage; };  // pair: two workgroups on a compute unit against one
    static constexpr Shape kShape[kGroupedShapeCount] = {{11.2f, 1.26f, 1, 1}, {10.0f, .625f, 1, 1}, {4.87f, .478f, 1, 1}, {2.78f, .393f, 1.26f, 1.74f}, {4.14f, .465f, 1.32f, 2.27f}};
    constexpr int kOrder[kGroupedShapeCount] = {2, 4, 0, 1, 3};  // (of equals the first)
    const float mean = (float)a.count / groups, stages = (float)((a.k + kTiledStage - 1) / kTiledStage);
    const float stream = (float)groups * a.n * a.k / 6.0e6f + 3.f;
    int best = 2;
    float least = INFINITY;
    for (int shape : kOrder) {
        const TiledShape& s = kGroupedShapes[shape];
        const float tiles = groups * fmaxf(1.f, mean / s.bm + .5f) * ((a.n + s.bn - 1) / s.bn), slots = (float)(kNumCU * s.per_cu);
        auto round_us = [&](float count) {
            const bool pair = count > kNumCU;
            return count <= 0 ? 0.f : kShape[shape].fixed * (pair ? kShape[shape].pair_fixed : 1.f) + stages * kShape[shape].stage * (pair ? kShape[shape].pair_stage : 1.f);
        };
        const float rounds = floorf(tiles / slots), t = fmaxf(rounds * round_us(slots) + round_us(tiles - rounds * slots), stream);
        if (t < least) {
            least = t;
            best = shape;
        }
    }
    return best;
}

// The tiled kernel on groups.
static int launch_grouped_tiles(const GroupedArgs& a, bool int8, int groups, hipStream_t stream) {
    const int shape = grouped_shape(a, groups);
    const TiledShape& s = kGroupedShapes[shape];
    const long grid = grouped_tiles_bound(a.count, a.experts, s.bm) * ((a.n + s.bn - 1) / s.bn);
    if (grid * s.threads > (long)UINT_MAX) return HFRK_BAD_SHAPE;
    TiledGroupedArgs t{};
    t.A = a.A;
    t.B = a.B;
    t.D = a.D;
    t.scale_a = a.scale_a;
    t.scale_b = a.scale_b;
    t.sa_stride = a.sa_stride;
    t.sb_stride = a.sb_stride;
    t.m = a.count;
    t.n = a.n;
    t.k = a.k;
    t.b_stride = a.b_stride;
    t.d_dtype = a.d_dtype;
    t.vec = a.n % 8 == 0 && (reinterpret_cast<uintptr_t>(a.D) & 15) == 0;
    t.tiles_m = ((a.count - 1) / groups + s.bm) / s.bm;  // of a group of the mean size: what the walk of the tiles and of k goes by
    t.tiles_n = (a.n + s.bn - 1) / s.bn;
    const int square = s.bm == s.bn ? 6 : 4;
    t.group_m = t.tiles_m < square ? t.tiles_m : square;
    t.splits = 1;
    t.stages_q = (a.k + kTiledStage - 1) / kTiledStage;
    turn_k(&t, s, false);
    t.offsets = a.offsets;
    t.rows = a.rows;
    t.expert_stride = a.expert_stride;
    t.sb_expert_stride = a.sb_expert_stride;
    t.count = a.count;
    t.a_rows = a.a_rows;
    t.experts = a.experts;
    return int8 ? launch_tiled_grouped_int8(t, shape, grid, stream) : launch_tiled_grouped_fp8(t, shape, grid, stream);
}

// Up to ten rows a group go to the rows kernel: its workgroup streams a weight for 16 rows at most (64 tokens on 2 of
// 8 experts of 28672 x 4096, 16 rows each: 213 us, tiles 182; 8 rows each 164 and 180; 128 on 6 of 64 of 2816 x 2048, 12 each, 76.9 and 75.3).
constexpr int kFewRowsPerGroup = 10;

template <bool INT8>
static int launch_grouped(const GroupedArgs& a, hipStream_t stream) {
    const int groups = a.experts < a.count ? a.experts : a.count;
    if (a.count / groups > kFewRowsPerGroup) return launch_grouped_tiles(a, INT8, groups, stream);
    const float active = a.experts * (1.f - powf(1.f - 1.f / a.experts, (float)a.count));  // groups that have rows, if all are as likely
    return launch_few_rows<INT8>(a, few_rows_kernel(a.n, a.k, fmaxf(active, 1.f), a.count / fmaxf(active, 1.f)), stream);
}

// One int8 weight that the skinny GEMM's kernels (below) do not take, as k is no multiple of 256 or its rows are too few to deal out: up to 16 rows the rows kernel,
// up to 32 the one with the smaller predicted time, more the tiled one, k in parts where that is worth clearing their counters (a launch of 2 us) and the caller
// gave memory for them.  Rows kernel and tiles at 8 / 17 / 32 rows, us: 4096 x 4112 6.7 / 7.8 / 9.0 and 12.2 / 13.2 / 15.3, 10000 x 5136 15.4 / 22.5 / 25.7 and
// 17.2 / 18.9 / 21.7, 28672 x 4112 29.3 / 39.1 / 46.3 and 30.4 / 32.3 / 35.2; the loss is 2304 x 5136 at 32 rows, 10.5 and 12.2.
constexpr int kDenseFewRows = 16;

static hfrk_tiled_plan int8_plan(int m, int n, int k, bool split, float* us) {
    hfrk_tiled_plan whole, parts;
    *us = make_tiled_plan(m, n, k, 1, &whole);
    const float shared = split ? make_tiled_plan(m, n, k, kTiledMaxSplits, &parts) + 2.f : *us;
    if (shared >= *us) return whole;
    *us = shared;
    return parts;
}

// The plan, or (false) that the rows kernel `few` is to run.
static bool int8_on_tiles(int m, int n, int k, bool split, hfrk_tiled_plan* p, FewRows* few) {
    const float tiles16 = (float)((m + 15) / 16);
    *few = few_rows_kernel(n, k, tiles16, m / tiles16);
    if (m <= kDenseFewRows) return false;
    float us;
    *p = int8_plan(m, n, k, split, &us);
    return m > 2 * kDenseFewRows || us < few->us;
}

static size_t int8_workspace_bytes(const hfrk_tiled_plan& p, int m, int n) { return tiled_plan_ws_bytes(p, m, n) + (size_t)tiled_plan_counters(p, m, n) * sizeof(int); }

__global__ void __launch_bounds__(256) clear_counters_kernel(int* counters, int count) {
    for (int i = blockIdx.x * 256 + threadIdx.x; i < count; i += gridDim.x * 256) counters[i] = 0;
}

// Up to 16 rows, and on weights above 8 MiB up to 32, a weight whose rows deal out evenly goes to the kernel of the skinny GEMM that gives every workgroup a band of
// rows (skinny_gemm_rows_impl.h, under the plan that fp8 codes have), against the kernels below, us: 6144 x 4096 at 1 / 4 / 16 / 17 / 32 rows 6.1 / 6.2 / 7.2 / 8.1 / 9.3
// and 7.9 / 8.0 / 9.1 / 11.3 / 12.0, 28672 x 4096 20.6 / 20.7 / 21.4 / 22.4 / 25.4 and 24.3 / 25.7 / 27.6 / 30.7 / 31.4, 4096 x 14336 at 1 / 4 / 16 / 17 rows 12.0 / 11.2 / 12.7 / 15.3 and
// 15.3 / 13.0 / 17.4 / 18.3, 2048 x 2048 3.6 / 3.6 / 4.0 / 5.7 / 6.2 and 4.1 / 4.3 / 4.7 / 4.8 / 4.8, 14336 x 512 at 17 rows 6.2 and 5.7.
constexpr int kBandRows = 32;
constexpr long kBandFromBytes = 8L << 20;  // above kDenseFewRows rows
constexpr int kBandRowsLongK = 24, kBandLongK = 8192;  // (4096 x 14336 at 32 rows: 18.0 to 20.6 us by what lies in the caches, on tiles 18.4 to 18.9; no other size was measured)

static bool int8_in_bands(const GroupedArgs& a, hfrk_gemm_plan* p) {
    if (a.count > kBandRows || (a.count > kDenseFewRows && (long)a.n * a.k <= kBandFromBytes) || (a.count > kBandRowsLongK && a.k > kBandLongK)) return false;
    if ((a.base && a.base_stride != 0 && a.base_stride != a.n) || (a.n % 4 == 0 && !a.vec)) return false;
    return ((long)a.n + 128) * a.b_stride + a.k < (1L << 31) && make_rows_plan(a.count, a.n, a.k, p) == HFRK_SUCCESS;
}

// From 17 rows to 64 with k = 2048 or 4096: the kernel whose waves split k between them and keep their rows in registers (skinny_gemm_ksplit.hip), against bands (up
// to 32 rows) or tiles, at 32 / 48 / 64 rows, us: 4096 x 4096 7.0 / 7.7 / 8.5 and 8.1 / 12.0 / 12.2, 28672 x 4096 22.9 / 24.5 / 26.3 and 25.5 / 32.7 / 34.0, 2048 x 2048
// 4.2 / 4.7 / 5.3 and 4.8 / 6.8 / 6.9; the loss is 14336 x 2048 at 33, 9.7 and 9.3.
static bool int8_in_window(const GroupedArgs& a, hfrk_gemm_plan* p) {
    if (a.count <= kDenseFewRows || a.count > HFRK_GEMM_MAX_M || (a.n % 4 == 0 && !a.vec)) return false;
    return ((long)a.n + 128) * a.b_stride + a.k < (1L << 31) && make_ksplit_plan(a.count, a.n, a.k, p) == HFRK_SUCCESS && p->slabs == 1;
}

// Both where they exist: bands where the 16-row tiles of the other leave a fifth of the compute units' rounds empty (at 24 rows 6144 x 4096, 1.5 rounds, 8.7 and 9.1
// us, 5120 x 4096, 1.25, 8.0 and 8.8; the other way round 10240 x 4096, 2.5, 12.3 and 11.7).
static bool int8_skinny(const GroupedArgs& a, hfrk_gemm_plan* p) {
    const long tiles = ((long)a.n + 15) / 16, rounds = (tiles + kNumCU - 1) / kNumCU;
    if (tiles > kNumCU && 4 * rounds * kNumCU >= 5 * tiles && int8_in_bands(a, p)) return true;
    return int8_in_window(a, p) || int8_in_bands(a, p);
}

// Under a plan of either kind.
static int launch_int8_skinny(const GroupedArgs& a, const hfrk_gemm_plan& p, hipStream_t stream) {
    GemmArgs g{};
    g.A = a.A;
    g.B = a.B;
    g.D = a.D;
    g.base = a.base;
    g.base_stride = a.base_stride;
    g.scale_a = a.scale_a;
    g.scale_b = a.scale_b;
    g.sa_stride = a.sa_stride;
    g.sb_stride = a.sb_stride;
    g.m = a.count;
    g.n = a.n;
    g.k = a.k;
    g.b_stride = a.b_stride;
    g.d_dtype = a.d_dtype;
    g.grid = p.grid;
    g.slabs = p.slabs;
    if (p.wn == -1) {
        g.panels = p.panels;
        g.units = p.panels * p.slabs;
        g.chunks_q = g.units / p.grid;
        g.chunks_r = g.units % p.grid;
        return launch_ksplit_int8_kernel(g, p.m_tiles, p.wk * 256, p.lds_bytes, stream);
    }
    set_rows_geometry(&g, p, false);
    return launch_rows_int8_kernel(g, p.ch, p.wk, p.lds_bytes, stream);
}

static int launch_int8(const GroupedArgs& a, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (!tiled_size_ok(a.count, a.n, a.k)) return HFRK_BAD_SHAPE;
    hfrk_gemm_plan skinny{};
    if (int8_skinny(a, &skinny)) return launch_int8_skinny(a, skinny, stream);
    hfrk_tiled_plan p{};
    FewRows few;
    bool tiles = int8_on_tiles(a.count, a.n, a.k, workspace != nullptr, &p, &few);
    if (tiles && int8_workspace_bytes(p, a.count, a.n) > workspace_bytes) tiles = int8_on_tiles(a.count, a.n, a.k, false, &p, &few);
    if (!tiles) return launch_few_rows<true>(a, few, stream);
    const size_t partials = tiled_plan_ws_bytes(p, a.count, a.n);
    int* const counters = p.splits > 1 ? reinterpret_cast<int*>(static_cast<uint8_t*>(workspace) + partials) : nullptr;
    if (counters) {
        const int count = (int)tiled_plan_counters(p, a.count, a.n);
        hipLaunchKernelGGL(clear_counters_kernel, dim3(count > 2048 ? 8 : 1), dim3(256), 0, stream, counters, count);
        HFRK_HIP_TRY(hipGetLastError());
    }
    return tiled_launch(a.A, a.B, false, a.D, a.base, a.base_stride, a.scale_a, a.sa_stride, a.scale_b, a.sb_stride, a.count, a.n, a.k, a.b_stride, a.d_dtype, p,
                        static_cast<float*>(workspace), partials, counters, stream, true);
}

static int grouped_run(GroupedArgs& a, int type, void* workspace, size_t workspace_bytes, hipStream_t stream) {
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
    if (!a.offsets) return launch_int8(a, workspace, workspace_bytes, stream);
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
    return hfrk::grouped_run(a, args->type, nullptr, 0, static_cast<hipStream_t>(stream));
}

size_t hfrk_int8_gemm_workspace_bytes(int m, int n, int k) {
    using namespace hfrk;
    hfrk_tiled_plan p{};
    hfrk_gemm_plan skinny{};
    FewRows few;
    if (!tiled_size_ok(m, n, k)) return 0;
    GroupedArgs a{};  // a call on side by side rows
    a.count = m;
    a.n = n;
    a.k = a.b_stride = k;
    a.vec = 1;
    if (int8_skinny(a, &skinny)) return 0;
    return int8_on_tiles(m, n, k, true, &p, &few) ? int8_workspace_bytes(p, m, n) : 0;
}

int hfrk_int8_gemm(const void* A, const void* B, void* D, const void* base, int base_stride, const float* scale_a, int sa_stride, const float* scale_b,
                   int sb_stride, int m, int n, int k, int b_stride, int d_dtype, void* workspace, size_t workspace_bytes, void* stream) {
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return HFRK_BAD_ALIGNMENT;
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
    return hfrk::grouped_run(a, HFRK_INT8, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

}  // extern "C"
