// Attention of many rows a key head over a paged cache: keys and values through LDS, for drafted trees and chains.
//
// The mathematics is that of tree_attention_kernel.h.  There every wave has its own tokens and holds them in registers; here the waves of a
// workgroup share them, each with 32 rows, and the products are of 32 x 32 with 16 in between:
//   S^T = K Q^T   keys are the A operand.  Row 16 t + 8 b + 4 h + r of a product is token 16 t + 8 h + 4 b + r, so that a lane's sixteen scores are
//                 those of eight tokens in a row for t = 0 and t = 1, from 16 t + 8 h on, h = lane / 32, all of query row lane % 32
//   O^T += V^T P  these, rounded to 16 bits, are the B operand for the 16 tokens of t; the A operand is V^T, turned when the tile is staged
// For 32 tokens and 32 rows of 128 columns there are 16 products of 32 cycles, 16 exponentials of 16, and what else there is.  A step of 32 tokens makes the next
// step's scores beside its own exponentials, so that the wave has products in flight while it has those.  Even so products and vector instructions are
// busy 45 and 44 % of a SIMD's cycles (16 trees of 64, 16384 tokens, 32/8 heads: 336 us, 0.8 PFLOP/s) and wait for each other more than they overlap.
//
// A tile is 64 tokens, two steps.  While one is computed on, the next is in flight to registers, 16 bytes a piece; behind the first step it is written to
// the other buffer in the order in which lanes read it as operands (fp8 converted, values turned in pairs of tokens), once for all waves:
//   keys    block (32 tokens, 16 columns): lane (row, h) at 16 * (32 h + (row ^ swizzle)); the swizzle spreads what neighbouring threads write over the banks
//   values  block (16 tokens, 32 columns): lane (row, h) at 16 * (32 h + row), a pair of tokens a word; row cc + 16 (j % 2) of block j / 2 is column
//           DP / 16 * cc + j
#pragma once

#include <type_traits>

#include "tree_attention_kernel.h"

namespace hfrk {

constexpr int kSharedTokens = 64;

typedef float v16f __attribute__((ext_vector_type(16)));

template <int DT>
__device__ __forceinline__ v16f mfma32(v4i a, v4i b, v16f c) {
    if constexpr (DT == HFRK_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// c plus the two 16-bit values of a word
template <int DT>
__device__ __forceinline__ float add2(int word, float c) {
    if constexpr (DT == HFRK_BF16) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, word), v2bf{(__bf16)1.f, (__bf16)1.f}, c, false);
    else return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2h, word), v2h{(_Float16)1.f, (_Float16)1.f}, c, false);
}

// The sum, or the largest, of the two lanes that hold the same query row.
template <typename OP>
__device__ __forceinline__ float of_both(float v, OP op) {
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(both[0]), __uint_as_float(both[1]));
}

// Every wave's LDS accesses are done and seen; requests to memory stay in flight (__syncthreads would wait for them).
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Marks (tree_attention_kernel.h) for products of 32 x 32.
template <int DT, int DP>
struct WideMarks {
    static constexpr int kBlocks = DP / 32, kWords = kBlocks / 2;  // 16 sums a block
    uint32_t rise[kWords] = {}, fall[kWords] = {};

    // seen: of 16 tokens each; values: in LDS, the lane's part of the first block's operand, those of the second 16 tokens behind all of the first's
    __device__ __forceinline__ void note(const uint32_t (&seen)[2], const v4i* values) {
#pragma unroll
        for (int w = 0; w < kWords; ++w)
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {
                v4i plus, minus;
                counted4<DT>(values[(i / 2 * kBlocks + 2 * w + i % 2) * kWave], plus, minus);
                const v4i sights = seen4<DT>(i < 2 ? seen[0] : seen[1]);
                const v16f up = mfma32<DT>(plus, sights, v16f(0.f)), down = mfma32<DT>(minus, sights, v16f(0.f));
                uint32_t u = 0, d = 0;
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    u |= (up[v] > 0.f ? 1u : 0u) << v;
                    d |= (down[v] > 0.f ? 1u : 0u) << v;
                }
                rise[w] |= u << i % 2 * 16;
                fall[w] |= d << i % 2 * 16;
            }
    }

    __device__ __forceinline__ void apply(v16f (&out)[kBlocks]) const {
        uint32_t any = 0;
#pragma unroll
        for (int w = 0; w < kWords; ++w) any |= rise[w] | fall[w];
        if (!__any(any != 0)) return;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                if (rise[b / 2] >> (b % 2 * 16 + v) & 1) out[b][v] += INFINITY;
                if (fall[b / 2] >> (b % 2 * 16 + v) & 1) out[b][v] -= INFINITY;
            }
    }
};

template <int DT, bool FP8, int DP, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, DP <= 128 ? 2 : 1) attention_shared_kernel(const AttentionArgs p) {
    constexpr int kThreads = 64 * WAVES;
    constexpr int kSteps = DP / 16;                  // products of 16 columns in K Q^T
    constexpr int kBlocks = DP / 32;                 // V^T's 32-row blocks
    constexpr int kCols = DP / 16, kSize = FP8 ? 1 : 2;
    constexpr int kGroups = 8 / WAVES;               // groups of eight tokens a wave stages, which share a page
    constexpr int kKeyUnits = DP / 64;               // pieces of their keys a lane has, of eight columns: a unit is 64 columns of all eight
    constexpr int kValueWords = kCols * kSize / 4;   // words of a value: kCols columns of two tokens a lane
    constexpr int kHalfBytes = kSharedTokens * DP * 2;  // keys, or values, of a tile
    constexpr int kTileBytes = 2 * kHalfBytes;
    __shared__ __align__(16) uint8_t tiles[2 * kTileBytes];   // [buffer][keys, values]
    __shared__ __align__(8) uint8_t exists[2][8];             // whether eight tokens have a page
    __shared__ uint32_t unsafe[2][WAVES];                     // whether a wave has staged an infinity or a NaN among drafted tokens' values

    const hfrk_attention_args& a = p.a;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
    const int item = blockIdx.x / a.kv_heads, head = blockIdx.x - item * a.kv_heads;
    const Part part = find_part(p, item);
    if (!part.any) return;
    const Sequence s = part.s;
    const int block0 = part.block * p.rows, row = block0 + wave * 32 + col, rows = s.count * p.group;
    const int drafted = s.drafted;

    const bool real = row < rows;
    const int row_token = row / p.group, member = row - row_token * p.group;
    const int seen_to = real ? drafted + row_token : -1;
    const uint8_t* const sees = static_cast<const uint8_t*>(a.mask) + (real ? (long)(s.first + row_token) * a.mask_stride : 0);
    v4i query[kSteps];
    {
        const uint16_t* const q = static_cast<const uint16_t*>(a.query) + (real ? (long)(s.first + row_token) * a.query_token_stride +
                                                                                  (long)(head * p.group + member) * a.query_head_stride : 0);
#pragma unroll
        for (int step = 0; step < kSteps; ++step) {
            const int d = 16 * step + 8 * h;
            query[step] = real && d < a.head_dim ? *reinterpret_cast<const v4i*>(q + d) : v4i{0, 0, 0, 0};
        }
    }
    const float scale = p.log2_scale * (FP8 && a.key_scale ? a.key_scale[head * a.key_scale_stride] : 1.f);

    // ---- staging
    const int32_t* const table = a.page_table + (long)part.b * a.table_stride;
    const uint8_t* const keys = static_cast<const uint8_t*>(a.key_cache) + (long)head * a.key_cache_head_stride * kSize;
    const uint8_t* const values = static_cast<const uint8_t*>(a.value_cache) + (long)head * a.value_cache_head_stride * kSize;
    // Where a group's tokens lie: the page's number is asked for a tile ahead of its use, and always, so that no wait for it takes in the requests of
    // keys and values behind it.
    struct Place {
        int asked, at, in_page;
    };
    typedef typename std::conditional<FP8, uint2, v4i>::type KeyPiece;
    KeyPiece key[kGroups][kKeyUnits];
    uint32_t value[kGroups][2][kValueWords];
    Place place[kGroups];
    int page[kGroups];        // of the tile that is to be requested, -1: none
    bool page_here[kGroups];  // whether the one that has been requested has one
    const int key_piece = (lane >> 4 & 1) * 4 + (lane & 3), key_token = (lane >> 5) * 4 + (lane >> 2 & 3);
    const int value_piece = lane & 15, value_pair = lane >> 4;
    const uint32_t key_lane = key_token * p.key_place_bytes;
    const uint32_t value_lane = 2 * value_pair * p.value_place_bytes + (value_piece * kCols < a.head_dim ? value_piece * kCols : 0) * kSize;
    auto group_token = [&](int n) { return 8 * (wave + WAVES * n); };  // the first of the wave's group n in the tile
    auto find_places = [&](int t0) {
#pragma unroll
        for (int n = 0; n < kGroups; ++n) {
            const int token = t0 + group_token(n);
            const uint32_t eights = (uint32_t)token >> 3;
            const int at = (int)(p.page_magic ? __umulhi(eights, p.page_magic) >> p.page_shift : eights >> p.page_shift);
            place[n] = {table[min(at, a.table_columns - 1)], at, token - at * a.page_size};
        }
    };
    auto settle = [&]() {
#pragma unroll
        for (int n = 0; n < kGroups; ++n) {
            const int number = __builtin_amdgcn_readfirstlane(place[n].asked);
            page[n] = place[n].at < a.table_columns && (uint32_t)number < (uint32_t)a.pages ? number : -1;
        }
    };
    auto request = [&]() {
#pragma unroll
        for (int n = 0; n < kGroups; ++n) {
            page_here[n] = page[n] >= 0;
            const uint64_t number = (uint32_t)max(page[n], 0);
            const uint8_t* const k_page = keys + (number * p.key_page_bytes + place[n].in_page * p.key_place_bytes);
            const uint8_t* const v_page = values + (number * p.value_page_bytes + place[n].in_page * p.value_place_bytes);
#pragma unroll
            for (int j = 0; j < kKeyUnits; ++j) {
                const int d = 64 * j + 8 * key_piece;  // (columns a head does not have are read elsewhere and cleared)
                key[n][j] = *reinterpret_cast<const KeyPiece*>(k_page + (key_lane + (d < a.head_dim ? d : 0) * kSize));
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint8_t* const from = v_page + (t * p.value_place_bytes + value_lane);
                if constexpr (kValueWords == 1) value[n][t][0] = *reinterpret_cast<const uint32_t*>(from);
                if constexpr (kValueWords == 2) *reinterpret_cast<uint2*>(value[n][t]) = *reinterpret_cast<const uint2*>(from);
                if constexpr (kValueWords >= 4) {
#pragma unroll
                    for (int w = 0; w < kValueWords; w += 4) *reinterpret_cast<uint4*>(value[n][t] + w) = *reinterpret_cast<const uint4*>(from + 4 * w);
                }
            }
        }
    };
    // Block 2 s + hh of eight columns; neighbouring threads write four blocks of four tokens.
    auto swizzle = [](int step, int hh) { return 4 * (2 * (step % 2) + hh); };
    auto put = [&](int buffer, int t0) {
        bool some = false;
#pragma unroll
        for (int n = 0; n < kGroups; ++n) {
            const int token8 = group_token(n);
            {
                const int w = token8 % 32 + key_token;  // of the half tile's 32
                const int r = w / 16 * 16 + w / 4 % 2 * 8 + w / 8 % 2 * 4 + w % 4;
                uint8_t* const to = tiles + buffer * kTileBytes + token8 / 32 * (kHalfBytes / 2);
#pragma unroll
                for (int j = 0; j < kKeyUnits; ++j) {
                    const int block = 8 * j + key_piece;
                    v4i x;
                    if constexpr (FP8) x = v4i{widen2<DT, false>(key[n][j].x), widen2<DT, true>(key[n][j].x), widen2<DT, false>(key[n][j].y), widen2<DT, true>(key[n][j].y)};
                    else x = key[n][j];
                    if (8 * block >= a.head_dim) x = v4i{0, 0, 0, 0};
                    *reinterpret_cast<v4i*>(to + (block / 2 * 64 + block % 2 * 32 + (r ^ swizzle(block / 2, block % 2))) * 16) = x;
                }
            }
            uint32_t keep = 0xffffffffu;  // tokens behind the end and without a page are cleared
            if (!page_here[n] || t0 + kSharedTokens > s.length) {
                const int left = page_here[n] ? s.length - (t0 + token8 + 2 * value_pair) : 0;
                keep = (left > 0 ? 0xffffu : 0u) | (left > 1 ? 0xffff0000u : 0u);
            }
            uint8_t* const to = tiles + buffer * kTileBytes + kHalfBytes + (token8 / 16 * kBlocks * 64 + token8 / 8 % 2 * 32 + value_piece) * 16 + value_pair * 4;
            uint32_t pairs[kCols];
#pragma unroll
            for (int f = 0; f < kCols; f += 2) {
                uint32_t even, odd;
                if constexpr (FP8) {
                    even = f % 4 == 0 ? widen2<DT, false>(value[n][0][f / 4]) : widen2<DT, true>(value[n][0][f / 4]);
                    odd = f % 4 == 0 ? widen2<DT, false>(value[n][1][f / 4]) : widen2<DT, true>(value[n][1][f / 4]);
                } else {
                    even = value[n][0][f / 2];
                    odd = value[n][1][f / 2];
                }
                pairs[f] = __builtin_amdgcn_perm(odd, even, 0x05040100u) & keep;
                pairs[f + 1] = __builtin_amdgcn_perm(odd, even, 0x07060302u) & keep;
                *reinterpret_cast<uint32_t*>(to + f / 2 * 1024) = pairs[f];
                *reinterpret_cast<uint32_t*>(to + f / 2 * 1024 + 256) = pairs[f + 1];
            }
            if (t0 + kSharedTokens > drafted) {
                uint32_t bad = 0;
#pragma unroll
                for (int f = 0; f < kCols; ++f) bad |= unbounded<DT>(pairs[f]);
                some |= __any(bad != 0) != 0;
            }
            if (lane == 0) exists[buffer][token8 / 8] = page_here[n];
        }
        if (lane == 0) unsafe[buffer][wave] = some;
    };

    // ---- the rows' state
    v16f out[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) out[b] = 0.f;
    float sum = 0.f, top = kNothing, bound = kNothing;  // bound: the raw score from which on the row's scale has to follow
    WideMarks<DT, DP> marks;

    int end = min(part.to, s.length);
    if (!a.mask) end = min(end, drafted + (min(block0 + p.rows, rows) - 1) / p.group + 1);  // a chain's rows see nothing behind the block's last token
    const int begin = part.from;
    const int steps = begin < end ? (end - begin + 31) / 32 : 0, tiles_here = (steps + 1) / 2;
    const int plain_to = min(drafted, s.length);  // tokens in front of it are seen by all, where they have a page
    if (steps > 0) {
        find_places(begin);
        settle();
        request();
        find_places(begin + kSharedTokens);
        settle();
        put(0, begin);
        if (tiles_here > 1) request();
        find_places(begin + 2 * kSharedTokens);
    }
    // The queries are here before the loop: waited for within it, a wait would take in the next tile's requests as well.
#pragma unroll
    for (int step = 0; step < kSteps; ++step) asm volatile("" : "+v"(query[step]));
    if (p.row_info && part.split == 0 && head == 0) {
        for (int r = threadIdx.x; r < p.rows && block0 + r < rows; r += kThreads)
            p.row_info[(long)s.first * p.group + block0 + r] = make_int4(part.slot, part.splits, r, 0);
    }

    // where the lane reads keys of even and odd blocks of 16 columns, in the present buffer
    const uint8_t *even_from = tiles + (h * 32 + (col ^ swizzle(0, h))) * 16, *odd_from = tiles + (h * 32 + (col ^ swizzle(1, h))) * 16;
    const uint8_t* value_from = tiles + kHalfBytes + lane * 16;
    int other = kTileBytes;  // from the present buffer to the other
    const auto load_keys = [&](int at, v4i (&k)[kSteps]) {
#pragma unroll
        for (int step = 0; step < kSteps; ++step) k[step] = *reinterpret_cast<const v4i*>((step % 2 ? odd_from : even_from) + at + step * 1024);
    };
    const auto score_keys = [&](const v4i (&k)[kSteps]) {
        v16f score = 0.f;
#pragma unroll
        for (int step = 0; step < kSteps; ++step) score = mfma32<DT>(k[step], query[step], score);
        return score;
    };
    v16f score;
    lds_barrier();
    {
        v4i k[kSteps];
        load_keys(0, k);
        score = score_keys(k);
    }
    constexpr int kAhead = kCols < 8 ? kCols : 8;  // blocks of values (of both halves of a step) read in front of the exponentials: all, up to 128 columns

    const auto step32 = [&](auto which, int buffer, int h0) {
        constexpr int half = decltype(which)::value;
        const uint32_t pages = *reinterpret_cast<const uint32_t*>(&exists[buffer][4 * half]);
        v4i turned[kAhead];
#pragma unroll
        for (int f = 0; f < kAhead; ++f) turned[f] = *reinterpret_cast<const v4i*>(value_from + (half * kCols + f) * 1024);
        bool unclean = false;
        if (h0 + 32 > plain_to || __builtin_amdgcn_readfirstlane(pages) != 0x01010101u) {
            uint32_t seen[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                seen[t] = sight(a, s, h0 + 16 * t + 8 * h, pages >> (16 * t + 8 * h) & 1u, seen_to, sees);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!(seen[t] >> j & 1)) score[8 * t + j] = -INFINITY;
            }
            // Rare: weights of zero do not keep an infinity or a NaN out of the sums.  They are noted for the rows that see their token, and taken out.
            uint32_t any = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) any |= unsafe[buffer][w];
            unclean = __builtin_amdgcn_readfirstlane(any) != 0;
            if (unclean) {
                marks.note(seen, reinterpret_cast<const v4i*>(value_from + half * kCols * 1024));
#pragma unroll
                for (int f = 0; f < kAhead; ++f) turned[f] = cleaned<DT>(turned[f]);
            }
        }
        // A row's scale follows its largest score when a lane has found one 2^8 above it, not with every step.
        float most = score[0];
#pragma unroll
        for (int j = 1; j < 16; ++j) most = fmaxf(most, score[j]);
        if (__any(most > bound)) {
            const float grown = fmaxf(top, of_both(most * scale, [](float x, float y) { return fmaxf(x, y); }) - kLift<DT>);
            const float shrink = __builtin_amdgcn_exp2f(top - grown);
            top = grown;
            bound = (grown + kHeadroom<DT>) / scale;
            sum *= shrink;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) out[b] *= shrink;
        }
        // The next step's keys: from the second half of a tile on they are in the next one, which all have written by now.  (All have read this one's
        // values too: behind the barrier its buffer is free, but where some blocks are read later.)
        if constexpr (half == 1) lds_barrier();
        v4i k[kSteps], weight[2];
        load_keys(half == 0 ? kHalfBytes / 2 : other, k);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = __builtin_amdgcn_exp2f(fmaf(score[8 * t + j], scale, -top));
            weight[t] = v4i{pack2<DT>(w[0], w[1]), pack2<DT>(w[2], w[3]), pack2<DT>(w[4], w[5]), pack2<DT>(w[6], w[7])};
#pragma unroll
            for (int q = 0; q < 4; ++q) sum = add2<DT>(weight[t][q], sum);
        }
        score = score_keys(k);
#pragma unroll
        for (int f = 0; f < kCols; ++f) {  // (16 tokens t = f / kBlocks, columns' block f % kBlocks)
            out[f % kBlocks] = mfma32<DT>(turned[f % kAhead], weight[f / kBlocks], out[f % kBlocks]);
            if (f + kAhead < kCols) {
                turned[f % kAhead] = *reinterpret_cast<const v4i*>(value_from + (half * kCols + f + kAhead) * 1024);
                if (unclean) turned[f % kAhead] = cleaned<DT>(turned[f % kAhead]);
            }
        }
    };
    for (int n = 0; n < tiles_here; ++n) {
        const int t0 = begin + kSharedTokens * n, buffer = n & 1;
        step32(std::integral_constant<int, 0>(), buffer, t0);
        settle();
        if (n + 1 < tiles_here) put(buffer ^ 1, t0 + kSharedTokens);
        if (n + 2 < tiles_here) request();
        find_places(t0 + 3 * kSharedTokens);
        if (2 * n + 1 >= steps) break;
        step32(std::integral_constant<int, 1>(), buffer, t0 + 32);
        if constexpr (kAhead < kCols) lds_barrier();
        even_from += other;
        odd_from += other;
        value_from += other;
        other = -other;
    }
    sum = of_both(sum, [](float x, float y) { return x + y; });
    marks.apply(out);
    const bool lost = top == kNothing;
    if (__any(lost)) {
        bool some;
        if constexpr (DP <= 64) {
            some = lost && sees_some(p, s, table, 8 * h, 16, seen_to, sees);
        } else {  // looked up again: held through the loop, the sequence took a register more of each lane (16 trees of 64: 344 -> 347 us; with heads of 64 there is room)
            const Sequence again = sequence(p, part.b);
            some = lost && real && sees_some(p, again, a.page_table + (long)part.b * a.table_stride, 8 * h, 16, again.drafted + row_token,
                                             static_cast<const uint8_t*>(a.mask) + (long)(again.first + row_token) * a.mask_stride);
        }
        top = fmaxf(top, of_both(some ? kSunk : kNothing, [](float x, float y) { return fmaxf(x, y); }));
    }

    // a lane has two runs of DP / 4 neighbouring columns of its row
    if (!real) return;
    const float value_scale = FP8 && a.value_scale ? a.value_scale[head * a.value_scale_stride] : 1.f;
    const float inv_out_scale = a.out_scale ? 1.f / a.out_scale[0] : 1.f;
    const long at = ((long)part.slot * a.kv_heads + head) * p.rows + (row - block0);
    if (part.splits > 1 && h == 0) p.partial_ml[at] = make_float2(top, sum);
#pragma unroll
    for (int run = 0; run < 2; ++run)
#pragma unroll
        for (int e = 0; e < 4 * kCols; e += 8) {
            const int d = kCols * (8 * run + 4 * h) + e;
            if (d >= a.head_dim) continue;
            float o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = (e + i) / kCols, j = (e + i) % kCols;
                o[i] = out[j / 2][4 * (run + 2 * (j % 2)) + r];
            }
            if (part.splits > 1) {
                float* const to = p.partial + at * a.head_dim + d;
                *reinterpret_cast<v4f*>(to) = v4f{o[0], o[1], o[2], o[3]};
                *reinterpret_cast<v4f*>(to + 4) = v4f{o[4], o[5], o[6], o[7]};
            } else {
                store_row<DT>(a, s.first + row_token, head * p.group + member, d, o, top, sum, value_scale, inv_out_scale);
            }
        }
}

template <int DP>
int launch_attention_shared(const AttentionArgs& p, int grid, hipStream_t stream) {
    const bool fp8 = p.a.cache_dtype == HFRK_FP8_E4M3FN;
#define HFRK_SHARED(DT, FP8)                                                                                                                    \
    do {                                                                                                                                        \
        if (p.rows == 128) hipLaunchKernelGGL((attention_shared_kernel<DT, FP8, DP, 4>), dim3(grid), dim3(256), 0, stream, p);                   \
        else if constexpr (DP < 256) hipLaunchKernelGGL((attention_shared_kernel<DT, FP8, DP, 8>), dim3(grid), dim3(512), 0, stream, p);         \
    } while (0)
    if (p.a.dtype == HFRK_BF16) {
        if (fp8) HFRK_SHARED(HFRK_BF16, true);
        else HFRK_SHARED(HFRK_BF16, false);
    } else {
        if (fp8) HFRK_SHARED(HFRK_F16, true);
        else HFRK_SHARED(HFRK_F16, false);
    }
#undef HFRK_SHARED
    HFRK_HIP_TRY(hipGetLastError());
    return HFRK_SUCCESS;
}

}  // namespace hfrk
