// Attention over a paged cache: checks, the choice of kernel, and the kernel that joins the parts of a row.
#include "tree_attention_kernel.h"

namespace hfrk {

extern template int launch_attention<64>(const AttentionArgs& p, int col_blocks, int grid, hipStream_t stream);
extern template int launch_attention<128>(const AttentionArgs& p, int col_blocks, int grid, hipStream_t stream);
extern template int launch_attention<256>(const AttentionArgs& p, int col_blocks, int grid, hipStream_t stream);
extern template int launch_attention_shared<64>(const AttentionArgs& p, int grid, hipStream_t stream);
extern template int launch_attention_shared<128>(const AttentionArgs& p, int grid, hipStream_t stream);
extern template int launch_attention_shared<256>(const AttentionArgs& p, int grid, hipStream_t stream);

// One wave per row of the result whose tokens were split: a lane has eight columns, lane groups take the splits in turn.  The order of
// the sums is fixed, so equal calls give equal bits.
template <int DT>
__global__ void __launch_bounds__(kAttentionThreads) attention_join_kernel(const AttentionArgs p) {
    const hfrk_attention_args& a = p.a;
    const int lane = threadIdx.x & (kWave - 1);
    const long index = (long)blockIdx.x * kAttentionWaves + (threadIdx.x >> 6);
    const long row = index / a.kv_heads;
    const int head = (int)(index - row * a.kv_heads);
    if (row >= (long)a.tokens * p.group) return;
    const int token = (int)(row / p.group), member = (int)(row - (long)token * p.group);
    if (a.starts && (token < a.starts[0] || token >= a.starts[a.seqs])) return;  // of no sequence
    const int4 info = p.row_info[row];
    const int first = info.x, splits = info.y;
    if (splits <= 1 || first < 0 || splits > p.slots - first || (uint32_t)info.z >= (uint32_t)p.rows) return;
    const long at = ((long)first * a.kv_heads + head) * p.rows + info.z, step = (long)a.kv_heads * p.rows;

    float most = -INFINITY;
    for (int s = lane; s < splits; s += kWave) most = fmaxf(most, p.partial_ml[at + s * step].x);
    most = wave_max(most);
    const int width = a.head_dim <= 128 ? 16 : 32, d = 8 * (lane & (width - 1));
    float total = 0.f, o[8] = {};
    for (int s = lane / width; s < splits; s += kWave / width) {
        const float2 ml = p.partial_ml[at + s * step];
        const float share = __builtin_amdgcn_exp2f(ml.x - most);
        total += share * ml.y;
        if (d < a.head_dim) {
            const v4f* const from = reinterpret_cast<const v4f*>(p.partial + (at + s * step) * a.head_dim + d);
            const v4f lo = from[0], hi = from[1];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[j] += share * lo[j];
                o[4 + j] += share * hi[j];
            }
        }
    }
    for (int by = width; by < kWave; by <<= 1) {
        total += __shfl_xor(total, by);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] += __shfl_xor(o[j], by);
    }
    if (lane >= width || d >= a.head_dim) return;
    const bool fp8 = a.cache_dtype == HFRK_FP8_E4M3FN;
    store_row<DT>(a, token, head * p.group + member, d, o, total, fp8 && a.value_scale ? a.value_scale[head * a.value_scale_stride] : 1.f,
                  a.out_scale ? 1.f / a.out_scale[0] : 1.f);
}

static int check(const hfrk_attention_args& a) {
    if (a.dtype != HFRK_F16 && a.dtype != HFRK_BF16) return HFRK_BAD_DTYPE;
    const bool fp8 = a.cache_dtype == HFRK_FP8_E4M3FN;
    if (!fp8 && a.cache_dtype != a.dtype) return HFRK_BAD_DTYPE;
    if (!fp8 && (a.key_scale || a.value_scale)) return HFRK_BAD_DTYPE;
    if (a.tokens < 0 || a.seqs < 0 || a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads != 0 || a.heads > 65536) return HFRK_BAD_SHAPE;
    if (a.head_dim < 16 || a.head_dim > 256 || a.head_dim % (fp8 || a.head_dim > 128 ? 16 : 8) != 0) return HFRK_BAD_SHAPE;
    if (a.page_size < 8 || a.page_size % 8 != 0 || a.pages < 0 || a.table_columns < 0) return HFRK_BAD_SHAPE;
    if ((long)a.table_columns * a.page_size > (1L << 30) || (long)a.tokens * a.heads > (1L << 28) || a.seqs > (1 << 20)) return HFRK_BAD_SHAPE;
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
    bool shared;
    int rows, work, grid, slots;
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
    d.shared = per > 32 && narrow(a.key_page_stride, a.key_place_stride, a.page_size, size) &&
               narrow(a.value_page_stride, a.value_place_stride, a.page_size, size);
    d.rows = per <= 16 ? 16 : per <= 32 || !d.shared ? 32 : per <= 128 || a.head_dim > 128 ? 128 : 256;
    d.work = d.shared ? 512 : 1024;
    const int rows = d.rows;
    const long blocks = (long)a.tokens * group / rows + a.seqs;
    const long tiles = ((long)a.table_columns * a.page_size + kTileTokens - 1) / kTileTokens;
    // sequences' splits are rounded up: one more than their share of the work each, and of those that are split at most twice their share
    const long items = d.work / a.kv_heads + 1 + blocks;
    d.grid = (int)(items * a.kv_heads);
    if (tiles > 1) {
        const long slots = 2 * (d.work / a.kv_heads + 1);
        d.slots = (int)(slots < blocks * tiles ? slots : blocks * tiles);
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
    p.work = d.work;
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
    const long waves = (long)a.tokens * a.heads;
    const dim3 grid((unsigned)((waves + kAttentionWaves - 1) / kAttentionWaves));
    if (a.dtype == HFRK_BF16) hipLaunchKernelGGL(attention_join_kernel<HFRK_BF16>, grid, dim3(kAttentionThreads), 0, s, p);
    else hipLaunchKernelGGL(attention_join_kernel<HFRK_F16>, grid, dim3(kAttentionThreads), 0, s, p);
    HFRK_HIP_TRY(hipGetLastError());
    return HFRK_SUCCESS;
}
