// Attention of many rows a key head over a paged cache: keys and values through LDS, for drafted trees and chains.
//
// The mathematics and the operands' order are those of tree_attention_kernel.h.  There every wave has its own tokens and holds them in registers; here
// RW waves share them, each with C blocks of 16 rows, and TW groups of such waves take the tile's 32-token halves in turn.  Products and
// exponentials bound it: for 32 tokens and 16 rows of 128 columns 17 products of 16 cycles, and for a lane's eight scores about 50 vector instructions,
// eight of them exponentials of 16 cycles; two waves a SIMD overlap the one with the other.
//
// A tile is 64 tokens.  While one is computed on, the next is in flight to registers, 16 bytes a piece; behind the products it is written to the other
// buffer, in the order in which lanes read it as matrix operands (fp8 converted, values turned in pairs of tokens), once for all waves:
//   keys    block (16 tokens, 32 columns): lane (token row i, column group g) at 16 * (16 g + (i ^ swizzle)); the swizzle spreads the pieces of one token,
//           which neighbouring threads write, over the banks
//   values  block (32 tokens, 16 columns kCols i + f): lane (i, token group g) at 16 * (16 g + i), a pair of tokens a word
#pragma once

#include <type_traits>

#include "tree_attention_kernel.h"

namespace hfrk {

constexpr int kSharedTokens = 64;

// Every wave's LDS accesses are done and seen; requests to memory stay in flight (__syncthreads would wait for them).
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int DT, bool FP8, int DP, int C, int RW, int TW>
__global__ void __launch_bounds__(64 * RW * TW) attention_shared_kernel(const AttentionArgs p) {
    constexpr int kThreads = 64 * RW * TW;
    constexpr int kSteps = DP / 32, kCols = DP / 16, kSize = FP8 ? 1 : 2;
    constexpr int kChunks = DP / 8;                                   // pieces of eight columns of a token
    constexpr int kKeyUnits = kSharedTokens * kChunks / kThreads;     // of keys a thread stages
    constexpr int kValueUnits = kSharedTokens / 2 * 16 / kThreads;    // of values: two tokens, kCols columns
    constexpr int kValueWords = kCols * kSize / 4;
    constexpr int kHalfBytes = kSharedTokens * DP * 2;                // keys, or values, of a tile
    static_assert(kThreads * kKeyUnits == kSharedTokens * kChunks && kThreads * kValueUnits == kSharedTokens * 8, "whole units a thread");
    static_assert(64 * RW * C * DP <= 4 * kHalfBytes || TW == 1, "the merge reuses the tiles");
    __shared__ __align__(16) uint8_t tiles[2][2][kHalfBytes];         // [buffer][keys, values]
    __shared__ int exists[2][kSharedTokens / 8];                      // whether eight tokens have a page
    __shared__ int unsafe[2][RW * TW];                                // whether a wave has staged an infinity or a NaN among drafted tokens' values
    __shared__ float statistics[RW][C * 16][2];

    const hfrk_attention_args& a = p.a;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const int row_wave = wave % RW, token_wave = wave / RW;
    const int item = blockIdx.x / a.kv_heads, head = blockIdx.x - item * a.kv_heads;
    const Part part = find_part(p, item);
    if (!part.any) return;
    const Sequence s = part.s;
    const int block0 = part.block * p.rows, row0 = block0 + row_wave * 16 * C, rows = s.count * p.group;
    const int drafted = s.drafted;

    v4i query[C][kSteps];
    int seen_to[C];
    const uint8_t* sees[C];
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

    // ---- staging: which pieces a thread brings; all of a wave's are of eight tokens at most that share a page
    const int32_t* const table = a.page_table + (long)part.b * a.table_stride;
    const uint8_t* const keys = static_cast<const uint8_t*>(a.key_cache) + (long)head * a.key_cache_head_stride * kSize;
    const uint8_t* const values = static_cast<const uint8_t*>(a.value_cache) + (long)head * a.value_cache_head_stride * kSize;
    // Where the wave's tokens lie: the page's number is asked for a tile ahead of its use, and always, so that no wait for it takes in the requests of
    // keys and values behind it.
    struct Place {
        int asked, at, in_page;
    };
    auto place_of = [&](int token) {  // the same token for the whole wave
        const uint32_t n = (uint32_t)token >> 3;
        const int at = (int)(p.page_magic ? __umulhi(n, p.page_magic) >> p.page_shift : n >> p.page_shift);
        return Place{table[min(at, a.table_columns - 1)], at, token - at * a.page_size};
    };
    auto page_of = [&](const Place& place) {  // -1: none
        const int page = __builtin_amdgcn_readfirstlane(place.asked);
        return place.at < a.table_columns && page >= 0 && page < a.pages ? page : -1;
    };
    typedef typename std::conditional<FP8, uint2, v4i>::type KeyPiece;
    KeyPiece key[kKeyUnits];
    uint32_t value[kValueUnits][2][kValueWords];
    Place key_place[kKeyUnits], value_place[kValueUnits];
    int key_page[kKeyUnits], value_page[kValueUnits];  // of the tile that is to be requested
    bool value_here[kValueUnits];                      // of the one that has been
    constexpr int kTokensAWave = kWave / kChunks > 0 ? kWave / kChunks : 1;  // key tokens a wave stages at a time
    static_assert(kWave % kChunks == 0 && kTokensAWave <= 8, "a wave's key pieces are of whole tokens within eight");
    const int key_chunk = lane % kChunks, key_row = lane / kChunks;
    const bool key_column = 8 * key_chunk < a.head_dim;
    const uint32_t key_lane = key_row * p.key_place_bytes + (key_column ? 8 * key_chunk : 0) * kSize;
    const bool value_column = col * kCols < a.head_dim;
    const uint32_t value_lane = 2 * g * p.value_place_bytes + (value_column ? col * kCols : 0) * kSize;
    auto key_token = [&](int j) { return (wave * kWave + kThreads * j) / kChunks; };
    auto value_token = [&](int j) { return 8 * (wave + RW * TW * j); };
    auto find_places = [&](int t0) {
#pragma unroll
        for (int j = 0; j < kKeyUnits; ++j) key_place[j] = place_of(t0 + key_token(j));
#pragma unroll
        for (int j = 0; j < kValueUnits; ++j) value_place[j] = place_of(t0 + value_token(j));
    };
    auto settle = [&]() {
#pragma unroll
        for (int j = 0; j < kKeyUnits; ++j) key_page[j] = page_of(key_place[j]);
#pragma unroll
        for (int j = 0; j < kValueUnits; ++j) value_page[j] = page_of(value_place[j]);
    };
    auto request = [&]() {
#pragma unroll
        for (int j = 0; j < kKeyUnits; ++j) {
            const uint8_t* const page = keys + (uint64_t)(uint32_t)max(key_page[j], 0) * p.key_page_bytes;
            key[j] = *reinterpret_cast<const KeyPiece*>(page + (key_place[j].in_page * p.key_place_bytes + key_lane));
        }
#pragma unroll
        for (int j = 0; j < kValueUnits; ++j) {
            value_here[j] = value_page[j] >= 0;
            const uint8_t* const page = values + (uint64_t)(uint32_t)max(value_page[j], 0) * p.value_page_bytes;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint8_t* const from = page + ((value_place[j].in_page + t) * p.value_place_bytes + value_lane);
                if constexpr (kValueWords == 1) value[j][t][0] = *reinterpret_cast<const uint32_t*>(from);
                if constexpr (kValueWords == 2) *reinterpret_cast<uint2*>(value[j][t]) = *reinterpret_cast<const uint2*>(from);
                if constexpr (kValueWords >= 4) {
#pragma unroll
                    for (int w = 0; w < kValueWords; w += 4) *reinterpret_cast<uint4*>(value[j][t] + w) = *reinterpret_cast<const uint4*>(from + 4 * w);
                }
            }
        }
    };
    auto swizzle = [](int step, int group) { return 4 * group + (DP == 64 ? 2 * step : step % 4); };
    auto put = [&](int buffer, int t0) {
        uint8_t* const k_to = tiles[buffer][0];
        uint8_t* const v_to = tiles[buffer][1];
#pragma unroll
        for (int j = 0; j < kKeyUnits; ++j) {
            const int token = key_token(j) + key_row, w = token % 32;
            const int t16 = token / 32 * 2 + w / 4 % 2, i = 4 * (w / 8) + w % 4, step = key_chunk / 4, group = key_chunk % 4;
            v4i x;
            if constexpr (FP8) x = v4i{widen2<DT, false>(key[j].x), widen2<DT, true>(key[j].x), widen2<DT, false>(key[j].y), widen2<DT, true>(key[j].y)};
            else x = key[j];
            if (!key_column) x = v4i{0, 0, 0, 0};
            *reinterpret_cast<v4i*>(k_to + ((t16 * kSteps + step) * 64 + group * 16 + (i ^ swizzle(step, group))) * 16) = x;
        }
        uint32_t bad = 0;
#pragma unroll
        for (int j = 0; j < kValueUnits; ++j) {
            const int token = value_token(j);
            const int left = s.length - (t0 + token + 2 * g);
            const uint32_t keep = value_here[j] ? (left > 0 ? 0xffffu : 0u) | (left > 1 ? 0xffff0000u : 0u) : 0u;
            uint8_t* const to = v_to + (token / 32 * kCols * 64 + token % 32 / 8 * 16 + col) * 16 + g * 4;
#pragma unroll
            for (int f = 0; f < kCols; f += 2) {
                uint32_t even, odd;
                if constexpr (FP8) {
                    even = f % 4 == 0 ? widen2<DT, false>(value[j][0][f / 4]) : widen2<DT, true>(value[j][0][f / 4]);
                    odd = f % 4 == 0 ? widen2<DT, false>(value[j][1][f / 4]) : widen2<DT, true>(value[j][1][f / 4]);
                } else {
                    even = value[j][0][f / 2];
                    odd = value[j][1][f / 2];
                }
                const uint32_t x = __builtin_amdgcn_perm(odd, even, 0x05040100u) & keep, y = __builtin_amdgcn_perm(odd, even, 0x07060302u) & keep;
                *reinterpret_cast<uint32_t*>(to + f * 1024) = x;
                *reinterpret_cast<uint32_t*>(to + (f + 1) * 1024) = y;
                if (t0 + kSharedTokens > drafted) bad |= unbounded<DT>(x) | unbounded<DT>(y);
            }
            if (lane == 0) exists[buffer][token / 8] = value_here[j];
        }
        const bool some = __any(bad != 0);
        if (lane == 0) unsafe[buffer][wave] = some;
    };

    constexpr int kAhead = 4;                   // blocks of values a wave has requested from LDS
    constexpr int kSwizzles = DP == 64 ? 2 : 4;
    int key_offset[kSwizzles];  // where a lane reads a block of keys, by its step
#pragma unroll
    for (int i = 0; i < kSwizzles; ++i) key_offset[i] = (g * 16 + (col ^ swizzle(i, g))) * 16;

    v4f out[C][kCols], sum[C];
    float top[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        top[c] = -INFINITY;
        sum[c] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int f = 0; f < kCols; ++f) out[c][f] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    constexpr int kOne = DT == HFRK_BF16 ? 0x3f803f80 : 0x3c003c00;
    const v4i ones = {kOne, kOne, kOne, kOne};

    const auto what_is_seen = [&](int first, bool page, uint32_t (&seen)[C]) { sight<C>(a, s, first, page, seen_to, sees, seen); };
    Marks<DT, DP, C> marks;
    int end = min(part.to * kTileTokens, s.length);
    if (!a.mask) end = min(end, drafted + (min(block0 + p.rows, rows) - 1) / p.group + 1);
    int t0 = part.from * kTileTokens;
    if (t0 < end) {
        find_places(t0);
        settle();
        request();
        find_places(t0 + kSharedTokens);
        settle();
        put(0, t0);
        if (t0 + kSharedTokens < end) request();
    }
    // The queries are here before the loop: waited for within it, a wait would take in the next tile's requests as well.
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int step = 0; step < kSteps; ++step) asm volatile("" : "+v"(query[c][step]));
    lds_barrier();
    int buffer = 0;
    for (; t0 < end; t0 += kSharedTokens, buffer ^= 1) {
        const int t1 = t0 + kSharedTokens, t2 = t1 + kSharedTokens;
        find_places(t2);
        const uint8_t* const k_from = tiles[buffer][0];
        const uint8_t* const v_from = tiles[buffer][1];
        if (t1 > drafted) {
            int any = 0;
#pragma unroll
            for (int w = 0; w < RW * TW; ++w) any |= unsafe[buffer][w];
            if (__builtin_amdgcn_readfirstlane(any) != 0) {
                // Rare: weights of zero do not keep an infinity or a NaN out of the sums.  They are noted for the rows that see their token, and taken out of
                // the tile.
                for (int half = token_wave; half < 2; half += TW) {
                    uint32_t seen[C];
                    what_is_seen(t0 + 32 * half + 8 * g, exists[buffer][4 * half + g] != 0, seen);
                    marks.note(seen, reinterpret_cast<const v4i*>(v_from) + half * kCols * 64 + lane);
                }
                lds_barrier();
                for (int i = threadIdx.x; i < kHalfBytes / 16; i += kThreads) {
                    v4i* const x = reinterpret_cast<v4i*>(tiles[buffer][1]) + i;
                    *x = Marks<DT, DP, C>::cleaned(*x);
                }
                lds_barrier();
            }
        }
#pragma unroll 1
        for (int half = token_wave; half < 2; half += TW) {
            const int h0 = t0 + 32 * half, mine = h0 + 8 * g;
            if (h0 >= end) break;
            v4f score[C][2];
#pragma unroll
            for (int c = 0; c < C; ++c) score[c][0] = score[c][1] = v4f{0.f, 0.f, 0.f, 0.f};
            const uint8_t* k_half[kSwizzles];
#pragma unroll
            for (int i = 0; i < kSwizzles; ++i) k_half[i] = k_from + half * (2 * kSteps * 1024) + key_offset[i];
            v4i k[2][kSteps];
#pragma unroll
            for (int step = 0; step < kSteps; ++step)
#pragma unroll
                for (int t = 0; t < 2; ++t) k[t][step] = *reinterpret_cast<const v4i*>(k_half[step % kSwizzles] + (t * kSteps + step) * 1024);
            __builtin_amdgcn_sched_barrier(0);  // all requests in front of the products, which otherwise wait for each by itself
#pragma unroll
            for (int step = 0; step < kSteps; ++step)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int c = 0; c < C; ++c) score[c][t] = mfma16<DT>(k[t][step], query[c][step], score[c][t]);

            // the first values are on their way while the weights are made
            const uint8_t* const v_half = v_from + half * (kCols * 1024) + lane * 16;
            v4i turned[kAhead];
#pragma unroll
            for (int f = 0; f < kAhead; ++f) turned[f] = *reinterpret_cast<const v4i*>(v_half + f * 1024);

            const bool here_page = exists[buffer][4 * half + g] != 0;
            if (h0 + 32 > drafted || __any(!here_page || mine + 8 > s.length)) {
                uint32_t seen[C];
                what_is_seen(mine, here_page, seen);
#pragma unroll
                for (int c = 0; c < C; ++c) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (!(seen[c] >> j & 1)) score[c][j / 4][j % 4] = -INFINITY;
                }
            }

            // A row's scale follows its largest score when a lane has found one 2^8 above it, not with every step.
            float most[C];
            bool grows = false;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                most[c] = score[c][0][0];
#pragma unroll
                for (int j = 1; j < 8; ++j) most[c] = fmaxf(most[c], score[c][j / 4][j % 4]);
                most[c] *= scale;
                grows |= most[c] > top[c] + kHeadroom;
            }
            if (__any(grows)) {
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const float grown = fmaxf(top[c], row_max(most[c]));
                    const float shrink = top[c] == grown ? 1.f : __builtin_amdgcn_exp2f(top[c] - grown);
                    top[c] = grown;
                    sum[c] *= shrink;
#pragma unroll
                    for (int f = 0; f < kCols; ++f) out[c][f] *= shrink;
                }
            }
            v4i weight[C];
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const float base = top[c] == -INFINITY ? 0.f : top[c];
                float w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = __builtin_amdgcn_exp2f(fmaf(score[c][j / 4][j % 4], scale, -base));
                weight[c] = v4i{pack2<DT>(w[0], w[1]), pack2<DT>(w[2], w[3]), pack2<DT>(w[4], w[5]), pack2<DT>(w[6], w[7])};
                sum[c] = mfma16<DT>(ones, weight[c], sum[c]);
            }
#pragma unroll
            for (int f = 0; f < kCols; ++f) {
#pragma unroll
                for (int c = 0; c < C; ++c) out[c][f] = mfma16<DT>(turned[f % kAhead], weight[c], out[c][f]);
                if (f + kAhead < kCols) turned[f % kAhead] = *reinterpret_cast<const v4i*>(v_half + (f + kAhead) * 1024);
            }
        }
        settle();
        if (t1 < end) put(buffer ^ 1, t1);
        if (t2 < end) request();
        lds_barrier();
    }

    if (p.row_info && part.split == 0 && head == 0) {
        for (int r = threadIdx.x; r < p.rows && block0 + r < rows; r += kThreads)
            p.row_info[(long)s.first * p.group + block0 + r] = make_int4(part.slot, part.splits, r, 0);
    }

    marks.apply(out);

    // ---- the token groups' parts of a row, then the result: a lane has DP / 4 neighbouring columns of its rows
    if constexpr (TW > 1) {
        v4f* const parts = reinterpret_cast<v4f*>(&tiles[0][0][0]);
        if (token_wave == 1) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                if (g == 0) {
                    statistics[row_wave][c * 16 + col][0] = top[c];
                    statistics[row_wave][c * 16 + col][1] = sum[c][0];
                }
#pragma unroll
                for (int f = 0; f < kCols; ++f) parts[((row_wave * C + c) * kCols + f) * 64 + lane] = out[c][f];
            }
        }
        lds_barrier();
        if (token_wave == 1) return;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const float other = statistics[row_wave][c * 16 + col][0], most = fmaxf(top[c], other);
            const float mine = top[c] == most ? 1.f : __builtin_amdgcn_exp2f(top[c] - most), its = other == most ? 1.f : __builtin_amdgcn_exp2f(other - most);
            sum[c][0] = mine * sum[c][0] + its * statistics[row_wave][c * 16 + col][1];
            top[c] = most;
#pragma unroll
            for (int f = 0; f < kCols; ++f) out[c][f] = mine * out[c][f] + its * parts[((row_wave * C + c) * kCols + f) * 64 + lane];
        }
    }
    const float value_scale = FP8 && a.value_scale ? a.value_scale[head * a.value_scale_stride] : 1.f;
    const float inv_out_scale = a.out_scale ? 1.f / a.out_scale[0] : 1.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int row = row0 + c * 16 + col;
        if (row >= rows) continue;
        const int token = row / p.group, member = row - token * p.group;
        const long at = ((long)part.slot * a.kv_heads + head) * p.rows + (row - block0);
        if (part.splits > 1 && g == 0) p.partial_ml[at] = make_float2(top[c], sum[c][0]);
#pragma unroll
        for (int e = 0; e < 4 * kCols; e += 8) {
            const int d = g * 4 * kCols + e;
            if (d >= a.head_dim) continue;
            float o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = out[c][(e + j) % kCols][(e + j) / kCols];
            if (part.splits > 1) {
                float* const to = p.partial + at * a.head_dim + d;
                *reinterpret_cast<v4f*>(to) = v4f{o[0], o[1], o[2], o[3]};
                *reinterpret_cast<v4f*>(to + 4) = v4f{o[4], o[5], o[6], o[7]};
            } else {
                store_row<DT>(a, s.first + token, head * p.group + member, d, o, sum[c][0], value_scale, inv_out_scale);
            }
        }
    }
}

template <int DP>
int launch_attention_shared(const AttentionArgs& p, int grid, hipStream_t stream) {
    const bool fp8 = p.a.cache_dtype == HFRK_FP8_E4M3FN;
#define HFRK_SHARED(DT, FP8)                                                                                                              \
    do {                                                                                                                                  \
        if (p.rows == 64) hipLaunchKernelGGL((attention_shared_kernel<DT, FP8, DP, 1, 4, 2>), dim3(grid), dim3(512), 0, stream, p);        \
        else if (p.rows == 128) hipLaunchKernelGGL((attention_shared_kernel<DT, FP8, DP, DP == 256 ? 1 : 2, DP == 256 ? 8 : 4, DP == 256 ? 1 : 2>), dim3(grid), dim3(512), 0, stream, p); \
        else if constexpr (DP < 256) hipLaunchKernelGGL((attention_shared_kernel<DT, FP8, DP, 2, 8, 1>), dim3(grid), dim3(512), 0, stream, p); \
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
