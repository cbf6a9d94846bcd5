// Attention of a step's queries over a paged cache: the kernel.
//
//   o_i = sum_j 2^(c s_ij - m_i) v_j / sum_j 2^(c s_ij - m_i),  s_ij = q_i . k_j,  c = scale * key_scale * log2(e)
//
// over the cached tokens j that row i sees, m_i the largest c s_ij so far or less by at most 8 (one pass: when it follows, what has been summed is
// scaled down); in fp16 7 below that, as its weights have to be held above 2^-25.
// A row is one drafted token and one of the query heads that share a key head, so a group of heads reads its keys and values once.
//
// Each wave takes 32 cached tokens at a time and C blocks of 16 rows, from memory to its own registers; keys go through its own part of LDS:
//   S^T = K Q^T   keys are the A operand.  Row r of the two 16-row products is token 8 (r / 4) + 4 t + r % 4, so that a lane's eight scores are those
//                 of eight tokens in a row, 8 g .. 8 g + 7 for lane group g = lane / 16, all of query row lane % 16
//   O^T += V^T P  these eight are, rounded to 16 bits, already the B operand of the second product.  Its A operand is V^T: a lane has loaded
//                 the same eight tokens' values of DP / 16 neighbouring columns, and turns that block within its own registers
//   l += 1 P      the sum of the weights, as rounded, by one more product with ones
// Scores, sums and statistics are fp32.  The weights are rounded to the query's 16-bit type (half a step of 2^-8 or 2^-11 each, and the same
// rounded weights make the sum, so that the rounding does not tilt the mean).  In fp16 they lie between 2^7, or more, for a row's largest and 2^15, so that
// one of 2^-32 of the largest still counts: with 1 to 2^8 a flat tail of 131071 tokens 2^25 below a first one was lost, 0.4 % of the sum.
//
// The next tokens' keys are requested before the present scores are made, their values behind the products: a wave has up to 16 KB (128 columns, 16
// bits) in flight, and bytes bound the kernel.  Values are widened and turned two columns at a time beside the products: held turned, they
// took the registers of a third wave (fp8: 64 x 2731 tokens in 83 us, so 77).  64 sequences of 2731 tokens, 8 key heads, 4 query heads each,
// 128 columns: 16 bits in 131 us, 5.5 TB/s, fp8 in 77 us, 4.6 TB/s.  Three workgroups a compute unit instead of two: 137 and 84 us.
#pragma once

#include "tree_attention.h"

namespace hfrk {

// A row's scale is set so that its largest weight is 2^lift, and follows when one is 2^8 above that.
template <int DT>
constexpr float kLift = DT == HFRK_F16 ? 7.f : 0.f;
template <int DT>
constexpr float kHeadroom = 8.f + kLift<DT>;
constexpr float kNothing = -1e38f;  // the scale of a row that has seen nothing; finite, so that nothing has to be told apart
constexpr float kSunk = -0.9e38f;   // of one that has seen scores of minus infinity only: more than nothing, less than all others

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

template <int DT>
__device__ __forceinline__ v4f mfma16(v4i a, v4i b, v4f c) {
    if constexpr (DT == HFRK_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

template <int DT>
__device__ __forceinline__ int pack2(float lo, float hi) {  // round to nearest even
    if constexpr (DT == HFRK_BF16) return __builtin_bit_cast(int, __builtin_convertvector(v2f{lo, hi}, v2bf));
    else return __builtin_bit_cast(int, __builtin_convertvector(v2f{lo, hi}, v2h));
}

// Two e4m3 values of a word's low or high half as 16-bit values; exact in both types.
template <int DT, bool HIGH>
__device__ __forceinline__ int widen2(int word) {
    if constexpr (DT == HFRK_BF16) return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, 1.f, HIGH));
    else return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.f, HIGH));
}

// The largest of the four lanes that hold the same query row.
__device__ __forceinline__ float row_max(float v) {
    const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
    const auto rows = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(rows[0]), __uint_as_float(rows[1]));
}

// Eight values of a row of the result: divided by the sum of the weights, times the values' scale; a row that saw nothing is zero, one that saw scores of
// minus infinity only has no sum to divide by and is NaN.
template <int DT>
__device__ __forceinline__ void store_row(const hfrk_attention_args& a, long token, int head, int d, const float (&o)[8], float top, float total,
                                          float value_scale, float inv_out_scale) {
    const float by = total != 0.f ? value_scale / total : top > kNothing ? NAN : 0.f;
    const long at = token * a.output_token_stride + head * a.output_head_stride + d;
    if (a.out_scale) {
        uint32_t w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            w[j] = cvt_pk_fp8_or_nan(o[4 * j] * by * inv_out_scale, o[4 * j + 1] * by * inv_out_scale, 0u, false);
            w[j] = cvt_pk_fp8_or_nan(o[4 * j + 2] * by * inv_out_scale, o[4 * j + 3] * by * inv_out_scale, w[j], true);
        }
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.output) + at) = make_uint2(w[0], w[1]);
    } else {
        *reinterpret_cast<v4i*>(static_cast<uint16_t*>(a.output) + at) =
            v4i{pack2<DT>(o[0] * by, o[1] * by), pack2<DT>(o[2] * by, o[3] * by), pack2<DT>(o[4] * by, o[5] * by), pack2<DT>(o[6] * by, o[7] * by)};
    }
}

// Of a pair of 16-bit values, those that are infinite or NaN: bit 15 of each half.  (Arithmetic on both halves at once, no conditions: as
// conditions the rare path below took all scalar registers.)
template <int DT>
__device__ __forceinline__ uint32_t unbounded(uint32_t pair) {
    constexpr uint32_t e = DT == HFRK_BF16 ? 0x7f807f80u : 0x7c007c00u;
    return (((pair & e) ^ e) + 0x7fff7fffu & 0x80008000u) ^ 0x80008000u;
}

// Those bits as whole halves.
__device__ __forceinline__ uint32_t halves(uint32_t bits) { return (bits << 1) - (bits >> 15); }

// Of four e4m3 values, those that are NaN: bit 7 of each byte.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t four) { return (((four & 0x7f7f7f7fu) ^ 0x7f7f7f7fu) + 0x7f7f7f7fu & 0x80808080u) ^ 0x80808080u; }

// Of the unbounded ones, those that are NaN or of the wanted sign (sign: 0 plus, 0x80008000 minus), as the value one.
template <int DT>
__device__ __forceinline__ uint32_t counted(uint32_t pair, uint32_t bits, uint32_t sign) {
    constexpr uint32_t f = DT == HFRK_BF16 ? 0x007f007fu : 0x03ff03ffu, one = DT == HFRK_BF16 ? 0x3f80u : 0x3c00u;
    const uint32_t nan = (pair & f) + 0x7fff7fffu;
    return (((nan | ~(pair ^ sign)) & bits) >> 15) * one;  // (`bits` has the halves' top bits only)
}

// Of the eight cached tokens from `first` on, those that a row sees: bit j token first + j.  page: they have one; seen_to: the last token the row of a
// chain sees; sees: the row of the mask.
__device__ __forceinline__ uint32_t sight(const hfrk_attention_args& a, const Sequence& s, int first, bool page, int seen_to, const uint8_t* sees) {
    const auto first_of_8 = [](int n) { return (1u << min(max(n, 0), 8)) - 1u; };
    const uint32_t here = page ? first_of_8(s.length - first) : 0u;
    if (!a.mask) return first_of_8(seen_to + 1 - first) & here;
    const int at = first - s.drafted;  // of the first token among the drafted ones
    const int known = min(s.count, a.mask_columns);
    uint32_t bits = 0;
    if (known > 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) bits |= min((uint32_t)sees[min(max(at + j, 0), known - 1)], 1u) << j;
    }
    return ((bits & first_of_8(known - at)) | first_of_8(-at)) & here;
}

// Whether a row sees a cached token that has a page, of the lane's eight from `first` on and those `step` behind them each time, in any part of its sequence (the
// first that is looked at, mostly).  For rows that have met no finite score, behind the loop: noted in it, it took registers that the loop does not have
// (16 trees of 64: 347 -> 351 us).
__device__ __forceinline__ bool sees_some(const AttentionArgs& p, const Sequence& s, const int32_t* table, int first, int step, int seen_to, const uint8_t* sees) {
    for (const int end = p.a.mask ? s.length : min(s.length, seen_to + 1); first < end; first += step) {
        if (sight(p.a, s, first, true, seen_to, sees) == 0) continue;
        const uint32_t eights = (uint32_t)first >> 3;
        const int at = (int)(p.page_magic ? __umulhi(eights, p.page_magic) >> p.page_shift : eights >> p.page_shift);
        if (at < p.a.table_columns && (uint32_t)table[at] < (uint32_t)p.a.pages) return true;
    }
    return false;
}

// Values without infinities and NaN.
template <int DT>
__device__ __forceinline__ v4i cleaned(v4i v) {
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] &= (int)~halves(unbounded<DT>((uint32_t)v[q]));
    return v;
}

// Infinities and NaN of an operand of V^T as ones, those of a sign and NaN.
template <int DT>
__device__ __forceinline__ void counted4(v4i v, v4i& plus, v4i& minus) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const uint32_t bits = unbounded<DT>((uint32_t)v[q]);
        plus[q] = (int)counted<DT>((uint32_t)v[q], bits, 0u);
        minus[q] = (int)counted<DT>((uint32_t)v[q], bits, 0x80008000u);
    }
}

// What is seen of eight tokens, as ones.
template <int DT>
__device__ __forceinline__ v4i seen4(uint32_t seen) {
    constexpr uint32_t one = DT == HFRK_BF16 ? 0x3f80u : 0x3c00u;
    v4i sights;
#pragma unroll
    for (int q = 0; q < 4; ++q) sights[q] = (int)(((seen >> 2 * q & 1u) | (seen >> (2 * q + 1) & 1u) << 16) * one);
    return sights;
}

// Infinities and NaN among drafted tokens' values: which of a lane's sums one of either sign has reached (a NaN counts as both), a bit for each.
template <int DT, int DP, int C>
struct Marks {
    static constexpr int kCols = DP / 16, kWords = (4 * kCols + 31) / 32;
    uint32_t rise[C][kWords] = {}, fall[C][kWords] = {};

    // `values`: in LDS, the lane's part of the operand of V^T's first 16-row block, the others 1 KB apart.  One block at a time, in a loop: unrolled, this
    // rare path takes the registers of the usual one.
    __device__ __forceinline__ void note(const uint32_t (&seen)[C], const v4i* values) {
#pragma unroll 1
        for (int f = 0; f < kCols; ++f) {
            v4i plus, minus;
            counted4<DT>(values[f * kWave], plus, minus);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const v4i sights = seen4<DT>(seen[c]);
                const v4f none = {0.f, 0.f, 0.f, 0.f};
                const v4f up = mfma16<DT>(plus, sights, none), down = mfma16<DT>(minus, sights, none);
#pragma unroll
                for (int r = 0; r < 4; ++r) {  // (a word holds 32 / kCols runs r of kCols bits)
                    rise[c][r * kCols / 32] |= (up[r] > 0.f ? 1u : 0u) << (r * kCols % 32 + f);
                    fall[c][r * kCols / 32] |= (down[r] > 0.f ? 1u : 0u) << (r * kCols % 32 + f);
                }
            }
        }
    }

    __device__ __forceinline__ void apply(v4f (&out)[C][kCols]) const {
        uint32_t any = 0;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int w = 0; w < kWords; ++w) any |= rise[c][w] | fall[c][w];
        if (!__any(any != 0)) return;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int f = 0; f < kCols; ++f)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int bit = r * kCols + f;
                    if (rise[c][bit / 32] >> bit % 32 & 1) out[c][f][r] += INFINITY;
                    if (fall[c][bit / 32] >> bit % 32 & 1) out[c][f][r] -= INFINITY;
                }
    }
};

// A wave's lanes read from its LDS what others of them have written: the LDS keeps their order, and so has the compiler to.
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// One wave's operands of 32 cached tokens.
template <int DP, bool FP8>
struct CachedTile {
    static constexpr int kWords = (FP8 ? DP / 16 : DP / 8) / 4;  // of a lane's columns of one token
    uint32_t key[8][kWords], value[8][kWords];
};

template <int DT, bool FP8, int DP, int C>
__global__ void __launch_bounds__(kWave * kDirectWaves, DP <= 128 ? 2 : 1) attention_kernel(const AttentionArgs p) {
    constexpr int kWaves = kDirectWaves, kThreads = kWave * kWaves, kAllTokens = kWaveTokens * kWaves;
    constexpr int kSteps = DP / 32;   // products of 32 columns in K Q^T
    constexpr int kCols = DP / 16;    // V^T's 16-row blocks, and the neighbouring columns a lane loads
    constexpr int kSize = FP8 ? 1 : 2;
    constexpr int kPad = DP + 4;
    typedef CachedTile<DP, FP8> Tile;
    __shared__ __align__(16) float merged[kWaves][16][kPad];
    __shared__ float statistics[kWaves][16][2];

    const hfrk_attention_args& a = p.a;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
    const int item = blockIdx.x / a.kv_heads, head = blockIdx.x - item * a.kv_heads;
    const Part part = find_part(p, item);
    if (!part.any) return;
    const Sequence s = part.s;
    const int row0 = part.block * p.rows, rows = s.count * p.group;
    const int drafted = s.drafted;

    // queries: lane group g has 8 columns of each product's 32
    v4i query[C][kSteps];
    int seen_to[C];      // chain: the last token this lane's row sees (-1: no row)
    const uint8_t* sees[C];  // tree: its row of the mask
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int row = row0 + c * 16 + col, token = row / p.group, member = row - token * p.group;
        const bool real = row < rows;
        seen_to[c] = real ? drafted + token : -1;
        sees[c] = static_cast<const uint8_t*>(a.mask) + (real ? (long)(s.first + token) * a.mask_stride : 0);
        const uint16_t* const q = static_cast<const uint16_t*>(a.query) + (real ? (long)(s.first + token) * a.query_token_stride +
                                                                                  (long)(head * p.group + member) * a.query_head_stride : 0);
#pragma unroll
        for (int step = 0; step < kSteps; ++step) {
            const int d = 32 * step + 8 * g;
            query[c][step] = real && d < a.head_dim ? *reinterpret_cast<const v4i*>(q + d) : v4i{0, 0, 0, 0};
        }
    }
    const float scale = p.log2_scale * (FP8 && a.key_scale ? a.key_scale[head * a.key_scale_stride] : 1.f);

    // A lane reads kCols columns of eight tokens, keys and values alike: whole rows side by side in 16 lanes.  (As operands of K Q^T, 16 rows side by side,
    // neighbouring lanes read 64 places apart, and a compute unit took requests at a quarter of the rate.)
    const int token8 = 8 * g;
    const bool column = col * kCols < a.head_dim;  // columns a head does not have are read elsewhere; keys are cleared there, values not stored
    const uint8_t* const keys = static_cast<const uint8_t*>(a.key_cache) + ((long)head * a.key_cache_head_stride + (column ? col * kCols : 0)) * kSize;
    const uint8_t* const values = static_cast<const uint8_t*>(a.value_cache) + ((long)head * a.value_cache_head_stride + (column ? col * kCols : 0)) * kSize;
    const int32_t* const table = a.page_table + (long)part.b * a.table_stride;
    auto index_of = [&](int token) {
        const uint32_t n = (uint32_t)token >> 3;
        return (int)(p.page_magic ? __umulhi(n, p.page_magic) >> p.page_shift : n >> p.page_shift);
    };
    auto page_of = [&](int t0) {  // of the lane's eight tokens; -1: none
        const int at = index_of(t0 + token8);
        const int page = table[min(at, a.table_columns - 1)];
        return at < a.table_columns && (uint32_t)page < (uint32_t)a.pages ? page : -1;
    };
    auto load = [&](uint32_t (&to)[8][Tile::kWords], const uint8_t* cache, long page_stride, long place_stride, int t0, int page) {
        const int token = t0 + token8, in_page = token - index_of(token) * a.page_size;
        const uint8_t* at = cache + ((long)max(page, 0) * page_stride + (long)in_page * place_stride) * kSize;
#pragma unroll
        for (int j = 0; j < 8; ++j, at += place_stride * kSize) {
            if constexpr (Tile::kWords == 1) to[j][0] = *reinterpret_cast<const uint32_t*>(at);
            if constexpr (Tile::kWords == 2) *reinterpret_cast<uint2*>(to[j]) = *reinterpret_cast<const uint2*>(at);
            if constexpr (Tile::kWords >= 4) {
#pragma unroll
                for (int w = 0; w < Tile::kWords; w += 4) *reinterpret_cast<uint4*>(to[j] + w) = *reinterpret_cast<const uint4*>(at + 4 * w);
            }
        }
    };
    auto load_keys = [&](Tile& tile, int t0, int page) { load(tile.key, keys, a.key_page_stride, a.key_place_stride, t0, page); };
    auto load_values = [&](Tile& tile, int t0, int page) { load(tile.value, values, a.value_page_stride, a.value_place_stride, t0, page); };
    // The wave's own LDS turns keys from rows to operands: token 8 g + j is row 4 g + j % 4 of product j / 4; pieces of eight columns change places by the row,
    // which spreads a product's rows over the banks.
    uint8_t* const own = reinterpret_cast<uint8_t*>(&merged[wave][0][0]);
    constexpr int kChunks = DP / 8;
    auto piece_at = [](int token, int row, int chunk) { return (token * kChunks + (chunk ^ (DP == 64 ? row / 2 : row))) * 16; };
    auto turn_keys = [&](const Tile& tile) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int token = token8 + j, row = 4 * g + j % 4;
            uint32_t x[kCols / 2];
#pragma unroll
            for (int w = 0; w < kCols / 2; ++w) {
                if constexpr (FP8) x[w] = w % 2 == 0 ? widen2<DT, false>(tile.key[j][w / 2]) : widen2<DT, true>(tile.key[j][w / 2]);
                else x[w] = tile.key[j][w];
                if (!column) x[w] = 0;
            }
            if constexpr (kCols == 4) {
                *reinterpret_cast<uint2*>(own + piece_at(token, row, col / 2) + col % 2 * 8) = make_uint2(x[0], x[1]);
            } else {
#pragma unroll
                for (int w = 0; w < kCols / 2; w += 4)
                    *reinterpret_cast<uint4*>(own + piece_at(token, row, col * (kCols / 8) + w / 4)) = make_uint4(x[w], x[w + 1], x[w + 2], x[w + 3]);
            }
        }
    };

    v4f out[C][kCols], sum[C];
    float top[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        top[c] = kNothing;
        sum[c] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int f = 0; f < kCols; ++f) out[c][f] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    constexpr int kOne = DT == HFRK_BF16 ? 0x3f803f80 : 0x3c003c00;
    const v4i ones = {kOne, kOne, kOne, kOne};

    Marks<DT, DP, C> marks;
    // a chain's rows see nothing behind the block's last token
    int end = min(part.to, s.length);
    if (!a.mask) end = min(end, drafted + (min(row0 + p.rows, rows) - 1) / p.group + 1);
    int t0 = part.from + wave * kWaveTokens;
    Tile tile;
    int now = -1, next = -1;
    if (t0 < end) {
        now = page_of(t0);
        load_keys(tile, t0, now);
        load_values(tile, t0, now);
        next = page_of(t0 + kAllTokens);
    }
    // The queries are here before the loop: waited for within it, a wait would take in the next tokens' requests as well.
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int step = 0; step < kSteps; ++step) asm volatile("" : "+v"(query[c][step]));
    for (; t0 < end; t0 += kAllTokens) {
        const int t1 = t0 + kAllTokens;
        const bool more = t1 < end;
        const int after = page_of(t1 + kAllTokens);  // (always: a wait for it alone)

        turn_keys(tile);
        wave_order();
        if (more) load_keys(tile, t1, next);
        v4f score[C][2];
#pragma unroll
        for (int c = 0; c < C; ++c) score[c][0] = score[c][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int step = 0; step < kSteps; ++step)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const v4i k = *reinterpret_cast<const v4i*>(own + piece_at(8 * (col >> 2) + 4 * t + (col & 3), col, 4 * step + g));
#pragma unroll
                for (int c = 0; c < C; ++c) score[c][t] = mfma16<DT>(k, query[c][step], score[c][t]);
            }

        // Tokens that some row does not see: drafted ones, those behind the end, those without a page.
        const bool lost = now < 0 || t0 + token8 + 7 >= s.length;
        const bool some = t0 + kWaveTokens > drafted || __any(lost);
        uint32_t seen[C];
        if (some) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                seen[c] = sight(a, s, t0 + token8, now >= 0, seen_to[c], sees[c]);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!(seen[c] >> j & 1)) score[c][j / 4][j % 4] = -INFINITY;
            }
        }

        v4i weight[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float most = score[c][0][0];
#pragma unroll
            for (int j = 1; j < 8; ++j) most = fmaxf(most, score[c][j / 4][j % 4]);
            most *= scale;
            // a row's scale follows its largest score when a lane has found one 2^8 above it, not with every step
            if (__any(most > top[c] + kHeadroom<DT>)) {
                const float grown = fmaxf(top[c], row_max(most) - kLift<DT>);
                const float shrink = __builtin_amdgcn_exp2f(top[c] - grown);
                top[c] = grown;
                sum[c] *= shrink;
#pragma unroll
                for (int f = 0; f < kCols; ++f) out[c][f] *= shrink;
            }
            float w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = __builtin_amdgcn_exp2f(fmaf(score[c][j / 4][j % 4], scale, -top[c]));
            weight[c] = v4i{pack2<DT>(w[0], w[1]), pack2<DT>(w[2], w[3]), pack2<DT>(w[4], w[5]), pack2<DT>(w[6], w[7])};
        }

        // V^T: word q of column f holds tokens 2q and 2q + 1
        const auto turn = [&](int f, v4i& even_column, v4i& odd_column) {  // columns f, f + 1
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t even, odd;
                if constexpr (FP8) {
                    even = f % 4 == 0 ? widen2<DT, false>(tile.value[2 * q][f / 4]) : widen2<DT, true>(tile.value[2 * q][f / 4]);
                    odd = f % 4 == 0 ? widen2<DT, false>(tile.value[2 * q + 1][f / 4]) : widen2<DT, true>(tile.value[2 * q + 1][f / 4]);
                } else {
                    even = tile.value[2 * q][f / 2];
                    odd = tile.value[2 * q + 1][f / 2];
                }
                even_column[q] = (int)__builtin_amdgcn_perm(odd, even, 0x05040100u);
                odd_column[q] = (int)__builtin_amdgcn_perm(odd, even, 0x07060302u);
            }
        };
        if (some) {
            // Weights of zero do not keep an infinity or a NaN out of the sums.  Memory behind the end and without a page is cleared; a drafted
            // token's own are noted for the rows that see it, and taken out.
            const int left = now < 0 ? 0 : min(max(s.length - (t0 + token8), 0), 8);
            uint32_t bad = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int w = 0; w < Tile::kWords; ++w) {
                    tile.value[j][w] = j < left ? tile.value[j][w] : 0u;
                    bad |= FP8 ? nan_bytes(tile.value[j][w]) : unbounded<DT>(tile.value[j][w]);
                }
            if (__any(bad != 0)) {
                v4i* const parked = reinterpret_cast<v4i*>(own) + lane;  // (the scores have been made: no keys are there any more)
#pragma unroll
                for (int f = 0; f < kCols; f += 2) {
                    v4i x, y;
                    turn(f, x, y);
                    parked[f * kWave] = x;
                    parked[(f + 1) * kWave] = y;
                }
                marks.note(seen, parked);
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int w = 0; w < Tile::kWords; ++w) {
                        uint32_t& x = tile.value[j][w];
                        if constexpr (FP8) x &= ~((nan_bytes(x) << 1) - (nan_bytes(x) >> 7));
                        else x &= ~halves(unbounded<DT>(x));
                    }
            }
        }

#pragma unroll
        for (int c = 0; c < C; ++c) sum[c] = mfma16<DT>(ones, weight[c], sum[c]);
#pragma unroll
        for (int f = 0; f < kCols; f += 2) {
            v4i x, y;
            turn(f, x, y);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                out[c][f] = mfma16<DT>(x, weight[c], out[c][f]);
                out[c][f + 1] = mfma16<DT>(y, weight[c], out[c][f + 1]);
            }
        }
        if (more) load_values(tile, t1, next);
        wave_order();
        now = next;
        next = after;
    }

    marks.apply(out);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const bool lost = top[c] == kNothing;
        if (__any(lost)) top[c] = fmaxf(top[c], row_max(lost && sees_some(p, s, table, token8, kWaveTokens, seen_to[c], sees[c]) ? kSunk : kNothing));
    }

    // The waves' parts of a row: scaled to the largest of their largest scores and added, 16 rows at a time.
    const float value_scale = FP8 && a.value_scale ? a.value_scale[head * a.value_scale_stride] : 1.f;
    const float inv_out_scale = a.out_scale ? 1.f / a.out_scale[0] : 1.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        if (row0 + c * 16 >= rows) break;  // (the same for the whole workgroup)
        if (c > 0) __syncthreads();
        if (g == 0) {
            statistics[wave][col][0] = top[c];
            statistics[wave][col][1] = sum[c][0];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int f = 0; f < kCols; f += 4)
                *reinterpret_cast<v4f*>(&merged[wave][col][(4 * g + r) * kCols + f]) = v4f{out[c][f][r], out[c][f + 1][r], out[c][f + 2][r], out[c][f + 3][r]};
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * (DP / 8); i += kThreads) {
            const int r = i / (DP / 8), d = 8 * (i - r * (DP / 8)), row = row0 + c * 16 + r;
            if (row >= rows || d >= a.head_dim) continue;
            float most = statistics[0][r][0];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) most = fmaxf(most, statistics[w][r][0]);
            float total = 0.f, o[8] = {};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float part_top = statistics[w][r][0];
                const float share = __builtin_amdgcn_exp2f(part_top - most);
                total += share * statistics[w][r][1];
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] += share * merged[w][r][d + j];
            }
            if (part.splits > 1) {
                const long at = ((long)part.slot * a.kv_heads + head) * p.rows + c * 16 + r;
                float* const to = p.partial + at * a.head_dim + d;
                *reinterpret_cast<v4f*>(to) = v4f{o[0], o[1], o[2], o[3]};
                *reinterpret_cast<v4f*>(to + 4) = v4f{o[4], o[5], o[6], o[7]};
                if (d == 0) p.partial_ml[at] = make_float2(most, total);
            } else {
                const int token = row / p.group, member = row - token * p.group;
                store_row<DT>(a, s.first + token, head * p.group + member, d, o, most, total, value_scale, inv_out_scale);
            }
        }
    }
    if (p.row_info && part.split == 0 && head == 0) {
        for (int r = threadIdx.x; r < p.rows && row0 + r < rows; r += kThreads)
            p.row_info[(long)s.first * p.group + row0 + r] = make_int4(part.slot - part.split, part.splits, r, 0);
    }
}

template <int DP>
int launch_attention(const AttentionArgs& p, int col_blocks, int grid, hipStream_t stream) {
    const bool fp8 = p.a.cache_dtype == HFRK_FP8_E4M3FN;
#define HFRK_ATTENTION(DT, FP8)                                                                                                             \
    do {                                                                                                                                    \
        if (col_blocks == 1) hipLaunchKernelGGL((attention_kernel<DT, FP8, DP, 1>), dim3(grid), dim3(kWave * kDirectWaves), 0, stream, p);      \
        else hipLaunchKernelGGL((attention_kernel<DT, FP8, DP, 2>), dim3(grid), dim3(kWave * kDirectWaves), 0, stream, p);                      \
    } while (0)
    if (p.a.dtype == HFRK_BF16) {
        if (fp8) HFRK_ATTENTION(HFRK_BF16, true);
        else HFRK_ATTENTION(HFRK_BF16, false);
    } else {
        if (fp8) HFRK_ATTENTION(HFRK_F16, true);
        else HFRK_ATTENTION(HFRK_F16, false);
    }
#undef HFRK_ATTENTION
    HFRK_HIP_TRY(hipGetLastError());
    return HFRK_SUCCESS;
}

}  // namespace hfrk
