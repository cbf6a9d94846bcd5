// Attention over a paged cache: checks, the choice of kernel, and the kernel that joins the parts of a row.
#include "tree_attention_kernel.h"

namespace hfrk {

extern template int launch_attention<64>(const AttentionArgs& p, int col_blocks, int grid, hipStream_t stream);
extern template int launch_attention<128>(const AttentionArgs& p, int col_blocks, int grid, hipStream_t stream);
extern template int launch_attention<256>(const AttentionArgs& p, int col_blocks, int grid, hipStream_t stream);
extern template int launch_attention_shared<64>(const AttentionArgs& p, int grid, hipStream_t stream);
extern template int launch_attention_shared<128>(const AttentionArgs& p, int grid, hipStream_t stream);
extern template int launch_attention_shared<256>(const AttentionArgs& p, int grid, hipStream_t stream);

// Joins the parts of the rows whose tokens were split.  A row's columns are eight a lane, side by side in 16 lanes (32 above 128 columns); PER such groups
// of lanes take a row's parts in turn: one (many rows), as many as a wave has, or those of a whole workgroup (few rows, many parts).  The order of the
// sums is fixed, so equal calls give equal bits.
constexpr int kJoinThreads = 256;

template <int DT, int WIDTH, int PER>
__global__ void __launch_bounds__(kJoinThreads) attention_join_kernel(const AttentionArgs p) {
    constexpr int kInWave = kWave / WIDTH, kGroups = kJoinThreads / WIDTH;
    static_assert(PER == 1 || PER == kInWave || PER == kGroups, "a row is a group's, a wave's or a workgroup's");
    __shared__ float parked[PER == kGroups ? kJoinThreads / kWave : 1][WIDTH][10];
    const hfrk_attention_args& a = p.a;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6, group = threadIdx.x / WIDTH;
    const long index = p.join_first + (long)blockIdx.x * (kGroups / PER) + group / PER;
    const long row = index / a.kv_heads;
    const int head = (int)(index - row * a.kv_heads);
    if (row >= (long)a.tokens * p.group) return;
    const int token = (int)(row / p.group), member = (int)(row - (long)token * p.group);
    const int4 info = p.row_info[row];
    if (a.starts && (token < a.starts[0] || token >= a.starts[a.seqs])) return;  // of no sequence
    const int first = info.x, splits = info.y;
    if (splits <= 1 || first < 0 || splits > p.slots - first || (uint32_t)info.z >= (uint32_t)p.rows) return;
    const long at = ((long)first * a.kv_heads + head) * p.rows + info.z, step = (long)a.kv_heads * p.rows;

    const int d = 8 * (lane & (WIDTH - 1));
    const bool column = d < a.head_dim;
    float top = kNothing, total = 0.f, o[8] = {};
    auto merge = [&](float other_top, float other_total, const float (&other)[8]) {
        const float most = fmaxf(top, other_top), mine = __builtin_amdgcn_exp2f(top - most), its = __builtin_amdgcn_exp2f(other_top - most);
        top = most;
        total = mine * total + its * other_total;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = mine * o[j] + its * other[j];
    };
#pragma unroll 4
    for (int s = group % PER; s < splits; s += PER) {
        const float2 ml = p.partial_ml[at + s * step];
        const v4f* const from = reinterpret_cast<const v4f*>(p.partial + (at + s * step) * a.head_dim + (column ? d : 0));
        const v4f lo = from[0], hi = from[1];
        const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        merge(ml.x, ml.y, x);
    }
    if constexpr (PER > 1) {
#pragma unroll
        for (int by = WIDTH; by < kWave; by <<= 1) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = __shfl_xor(o[j], by);
            merge(__shfl_xor(top, by), __shfl_xor(total, by), x);
        }
    }
    if constexpr (PER == kGroups) {
        if (lane < WIDTH) {
            float* const to = parked[wave][lane];
#pragma unroll
            for (int j = 0; j < 8; ++j) to[j] = o[j];
            to[8] = top;
            to[9] = total;
        }
        __syncthreads();
        if (wave > 0 || lane >= WIDTH) return;
#pragma unroll
        for (int w = 1; w < kJoinThreads / kWave; ++w) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = parked[w][lane][j];
            merge(parked[w][lane][8], parked[w][lane][9], x);
        }
    }
    if (!column || (PER > 1 && lane >= WIDTH)) return;
    const bool fp8 = a.cache_dtype == HFRK_FP8_E4M3FN;
    store_row<DT>(a, token, head * p.group + member, d, o, top, total, fp8 && a.value_scale ? a.value_scale[head * a.value_scale_stride] : 1.f,
                  a.out_scale ? 1.f / a.out_scale[0] : 1.f);
}

template <int DT, int WIDTH>
static int launch_join(AttentionArgs p, hipStream_t stream) {
    constexpr int kGroups = kJoinThreads / WIDTH;
    const long rows = (long)p.a.tokens * p.a.heads;
    // A wave a row from one wave per compute unit's SIMD on, a group a row from four waves on: below, more lanes a row find room beside each other.
    const int per = rows < 4 * kNumCU ? kGroups : rows < 16 * kNumCU ? kWave / WIDTH : 1;
    const dim3 threads(kJoinThreads);
    const long most = (1L << 23) * kGroups / per;  // of a launch, whose threads are counted in 32 bits
    for (; rows - p.join_first > most; p.join_first += most) {  // (so many rows have a group each)
        hipLaunchKernelGGL((attention_join_kernel<DT, WIDTH, 1>), dim3(1 << 23), threads, 0, stream, p);
        HFRK_HIP_TRY(hipGetLastError());
    }
    const dim3 grid((unsigned)(((rows - p.join_first) * per + kGroups - 1) / kGroups));
    if (per == kGroups) hipLaunchKernelGGL((attention_join_kernel<DT, WIDTH, kGroups>), grid, threads, 0, stream, p);
    else if (per > 1) hipLaunchKernelGGL((attention_join_kernel<DT, WIDTH, kWave / WIDTH>), grid, threads, 0, stream, p);
    else hipLaunchKernelGGL((attention_join_kernel<DT, WIDTH, 1>), grid, threads, 0, stream, p);
    HFRK_HIP_TRY(hipGetLastError());
    return HFRK_SUCCESS;
}

static int check(const hfrk_attention_args& a) {
    if (a.dtype != HFRK_F16 && a.dtype != HFRK_BF16) return HFRK_BAD_DTYPE;
    const bool fp8 = a.cache_dtype == HFRK_FP8_E4M3FN;
    if (!fp8 && a.cache_dtype != a.dtype) return HFRK_BAD_DTYPE;
    if (!fp8 && (a.key_scale || a.value_scale)) return HFRK_BAD_DTYPE;
    if (a.tokens < 0 || a.seqs < 0 || a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads != 0 || a.heads > 65536) return HFRK_BAD_SHAPE;
    if (a.head_dim < 16 || a.head_dim > 256 || a.head_dim % (fp8 || a.head_dim > 128 ? 16 : 8) != 0) return HFRK_BAD_SHAPE;
    if (a.page_size < 8 || a.page_size % 8 != 0 || a.pages < 0 || a.table_columns < 0) return HFRK_BAD_SHAPE;
    if ((long)a.table_columns * a.page_size > (1L << 27) || (long)a.tokens * a.heads > (1L << 28) || a.seqs > (1 << 20)) return HFRK_BAD_SHAPE;
    // (row blocks times tiles, summed over sequences, stay below 2^32)
    if (!(a.scale > 0.f)) return HFRK_BAD_SHAPE;
    if (a.tokens == 0) return HFRK_SUCCESS;
    if (a.seqs < 1 || (!a.starts && a.tokens % a.seqs != 0)) return HFRK_BAD_SHAPE;
    if (a.pages < 1 || a.table_columns < 1) return HFRK_BAD_SHAPE;
    if (!a.query || !a.output || !a.key_cache || !a.value_cache || !a.page_table || !a.lengths) return HFRK_BAD_SHAPE;
    if (a.mask && a.mask_columns < 0) return HFRK_BAD_SHAPE;
    const int64_t piece = fp8 ? 16 : 8;
    if ((reinterpret_cast<uintptr_t>(a.query) | reinterpret_cast<uintptr_t>(a.key_cache) | reinterpret_cast<uintptr_t>(a.value_cache)) & 15) return HFRK_BAD_ALIGNMENT;
    if (reinterpret_cast<uintptr_t>(a.output) & (a.out_scale ? 7 : 15)) return HFRK_BAD_ALIGNMENT;
    if ((a.query_token_stride | a.query_head_stride | a.output_token_stride | a.output_head_stride) & 7) return HFRK_BAD_ALIGNMENT;
    if ((a.key_page_stride | a.key_place_stride | a.key_cache_head_stride | a.value_page_stride | a.value_place_stride | a.value_cache_head_stride) & (piece - 1))
        return HFRK_BAD_ALIGNMENT;
    return HFRK_SUCCESS;
}

// Rows of a block, the work list's bounds and the workspace, from what the host knows: sizes, not lengths.
struct Decomposition {
    bool shared, fits;
    int rows, tile, work, shares, grid, slots;
    size_t partial, ml, info;  // bytes
};

// Whether 32 bits hold a cache's strides and offsets in a page in bytes, as the kernels with LDS take them.
static bool narrow(int64_t page, int64_t place, int page_size, int size) {
    return page >= 0 && place >= 0 && page * size < (1LL << 32) && place * size * page_size < (1LL << 31);
}

static Decomposition decompose(const hfrk_attention_args& a) {
    Decomposition d = {};
    const int group = a.heads / a.kv_heads;
    const long per = (a.tokens + a.seqs - 1) / a.seqs * (long)group;  // rows of a sequence, on average
    const int size = a.cache_dtype == HFRK_FP8_E4M3FN ? 1 : 2;
    // With little work a workgroup has a tile or two, and what counts is how soon it has done one: the direct kernel, though its blocks of 32 rows read keys
    // more often.  From tiles of about 24 a compute unit on (4 where heads of more than 128 columns leave room for one workgroup) sharing pays, us:
    //     sequences x rows x tokens   4 x 48 x 2000   4 x 108 x 4000   8 x 108 x 2500   1 x 4096 x 1024   16 x 48 x 2731
    //     tiles a compute unit             8               22               23               33                30 (bf16, 128 columns)
    //     direct                         23.3             34.3             39.7             47.7              47.1
    //     shared                         24.4             37.3             38.2             50.5              44.3
    // (fp8: 20.7 and 25.1, 31.1 and 34.9, 34.9 and 35.8, 40.7 and 51.3.)  The host knows the table's columns, not the lengths.
    const long few = ((long)a.tokens * group / 32 + a.seqs) * (((long)a.table_columns * a.page_size + 127) / 128) * a.kv_heads;
    d.shared = per > 32 && few > (a.head_dim > 128 ? 4 : 24) * kNumCU && narrow(a.key_page_stride, a.key_place_stride, a.page_size, size) &&
               narrow(a.value_page_stride, a.value_place_stride, a.page_size, size);
    // A block of rows reads its keys once, so it is as large as the rows fill: 64 sequences x 2731 tokens, 8 key heads, 128 columns, us
    //     rows a sequence           32 fp8   64   64 fp8   128   256   400
    //     16 a block, direct           111
    //     32 a block, direct            84  199      119
    //     128 a block, shared          138  154      127   164   288   492
    //     256 a block, shared               217      195   229   262   441
    d.rows = per <= 16 ? 16 : per <= 32 || !d.shared ? 32 : per <= 128 || a.head_dim > 128 ? 128 : 256;
    d.tile = d.shared ? 128 : kWaveTokens * kDirectWaves;
    // (256 rows are eight waves, and heads of more than 128 columns fill the registers: one such workgroup a compute unit)
    d.work = d.rows == 256 || a.head_dim > 128 ? kNumCU : 2 * kNumCU;
    const int rows = d.rows;
    const long blocks = (long)a.tokens * group / rows + a.seqs;
    const long tiles = ((long)a.table_columns * a.page_size + d.tile - 1) / d.tile;
    // Workgroups take the whole's share or a part of it (find_part).  Splits are rounded up: one more than that a block, and of those that are split at
    // most twice as many.
    d.shares = a.seqs > 1 ? 2 : 1;
    const long most = (long)d.shares * (d.work / a.kv_heads > 1 ? d.work / a.kv_heads : 1), items = most + blocks < blocks * tiles ? most + blocks : blocks * (tiles > 0 ? tiles : 1);
    // Every workgroup makes the list of work from all sequences: 0.25, 3.1 and 50 ms for 1024, 4096 and 16384 sequences of 16 tokens, 8 key heads, where the last
    // is 2^31 workgroups times sequences.  (1024 sequences of 1000 to 2000 tokens, 1.23 ms, are at the rate of their bytes.)  At 2^36 a call would take
    // 1.6 s; it is refused from there on, as it would soon look as if it hung.
    // (A launch's threads are counted in 32 bits; more run as the rest, without an error.)
    d.fits = blocks * tiles < (1L << 31) && items * a.kv_heads * (rows == 256 ? 512 : 256) < (1L << 32) && items * a.kv_heads * a.seqs <= (1L << 36);
    d.grid = (int)(items * a.kv_heads);
    if (tiles > 1) {
        d.slots = (int)(2 * most < blocks * tiles ? 2 * most : blocks * tiles);
        d.partial = (size_t)d.slots * a.kv_heads * rows * a.head_dim * sizeof(float);
        d.ml = (size_t)d.slots * a.kv_heads * rows * sizeof(float2);
        d.info = (size_t)a.tokens * group * sizeof(int4);
    }
    return d;
}

}  // namespace hfrk

extern "C" size_t hfrk_tree_attention_workspace_bytes(const hfrk_attention_args* args) {
    using namespace hfrk;
    if (!args || check(*args) != HFRK_SUCCESS || args->tokens == 0) return 0;
    const Decomposition d = decompose(*args);
    return d.partial + d.info + d.ml;
}

extern "C" int hfrk_tree_attention(const hfrk_attention_args* args, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace hfrk;
    if (!args) return HFRK_BAD_SHAPE;
    const int status = check(*args);
    if (status != HFRK_SUCCESS || args->tokens == 0) return status;
    AttentionArgs p = {};
    p.a = *args;
    const hfrk_attention_args& a = p.a;
    const Decomposition d = decompose(a);
    if (!d.fits) return HFRK_BAD_SHAPE;
    if (d.slots > 0) {
        if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15)) return HFRK_BAD_ALIGNMENT;
        if (workspace_bytes < d.partial + d.info + d.ml) return HFRK_EXCEEDS_SCRATCH;
        uint8_t* const at = static_cast<uint8_t*>(workspace);
        p.partial = reinterpret_cast<float*>(at);
        p.row_info = reinterpret_cast<int4*>(at + d.partial);
        p.partial_ml = reinterpret_cast<float2*>(at + d.partial + d.info);
    }
    p.log2_scale = a.scale * 1.4426950408889634f;
    p.group = a.heads / a.kv_heads;
    p.rows = d.rows;
    p.tile = d.tile;
    p.work = d.work;
    p.shares = d.shares;
    p.slots = d.slots;
    const uint32_t size = a.cache_dtype == HFRK_FP8_E4M3FN ? 1 : 2;
    p.key_page_bytes = (uint32_t)a.key_page_stride * size;
    p.key_place_bytes = (uint32_t)a.key_place_stride * size;
    p.value_page_bytes = (uint32_t)a.value_page_stride * size;
    p.value_place_bytes = (uint32_t)a.value_place_stride * size;
    // n / m for n < 2^28, m = page_size / 8: with 2^(l-1) < m <= 2^l, ceil(2^(28+l) / m) is exact enough and has at most 29 bits
    const uint32_t m = (uint32_t)a.page_size / 8;
    int l = 0;
    while ((1u << l) < m) ++l;
    if ((1u << l) == m) {
        p.page_shift = l;
    } else {
        p.page_magic = (uint32_t)(((1ull << (28 + l)) + m - 1) / m) << 3;
        p.page_shift = l - 1;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    int launched;
    if (d.shared) {
        launched = a.head_dim <= 64 ? launch_attention_shared<64>(p, d.grid, s)
                   : a.head_dim <= 128 ? launch_attention_shared<128>(p, d.grid, s) : launch_attention_shared<256>(p, d.grid, s);
    } else {
        launched = a.head_dim <= 64 ? launch_attention<64>(p, d.rows / 16, d.grid, s)
                   : a.head_dim <= 128 ? launch_attention<128>(p, d.rows / 16, d.grid, s) : launch_attention<256>(p, d.rows / 16, d.grid, s);
    }
    if (launched != HFRK_SUCCESS || d.slots == 0) return launched;
    if (a.dtype == HFRK_BF16) return a.head_dim <= 128 ? launch_join<HFRK_BF16, 16>(p, s) : launch_join<HFRK_BF16, 32>(p, s);
    return a.head_dim <= 128 ? launch_join<HFRK_F16, 16>(p, s) : launch_join<HFRK_F16, 32>(p, s);
}
