// Attention of many rows a key head over a paged cache: keys and values through LDS, for drafted trees and chains.
//
// The mathematics and the operands' order are those of tree_attention_kernel.h.  There every wave has its own tokens and holds them in registers; here
// eight waves of C blocks of 16 rows share them.  Products and exponentials bound it: for 32 tokens and 16 rows of 128 columns 17 products of 16
// cycles, and for a lane's eight scores about 40 vector instructions, eight of them exponentials of 16 cycles.  Waves i and i + 4 share a SIMD: in one
// phase the first four have their products while the others have their exponentials, in the next the other way round, with a barrier between.
// (All in step, the same work took the sum of the two: 400 us instead of TODO for trees of 64 tokens over 16 caches of 16384.)
//
// A tile is 64 tokens.  While one is computed on, the next is in flight to registers, 16 bytes a piece; in a phase of exponentials it is written to
// the other buffer, in the order in which lanes read it as matrix operands (fp8 converted, values turned in pairs of tokens), once for all waves:
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

constexpr int kSharedWaves = 8;

template <int DT, bool FP8, int DP, int C>
__global__ void __launch_bounds__(64 * kSharedWaves) attention_shared_kernel(const AttentionArgs p) {
    constexpr int kThreads = 64 * kSharedWaves;
    constexpr int kSteps = DP / 32, kCols = DP / 16, kSize = FP8 ? 1 : 2;
    constexpr int kChunks = DP / 8;                                   // pieces of eight columns of a token
    constexpr int kKeyUnits = kSharedTokens * kChunks / kThreads;     // of keys a thread stages
    constexpr int kValueUnits = kSharedTokens / 2 * 16 / kThreads;    // of values: two tokens, kCols columns each
    constexpr int kValueWords = kCols * kSize / 4;
    constexpr int kHalfBytes = kSharedTokens * DP * 2;                // keys, or values, of a tile
    static_assert(kThreads * kKeyUnits == kSharedTokens * kChunks && kThreads * kValueUnits == kSharedTokens * 8, "whole units a thread");
    __shared__ __align__(16) uint8_t tiles[2][2][kHalfBytes];         // [buffer][keys, values]
    __shared__ int exists[2][kSharedTokens / 8];                      // whether eight tokens have a page
    __shared__ int unsafe[2][kSharedWaves];                                // whether a wave has staged an infinity or a NaN among drafted tokens' values

    const hfrk_attention_args& a = p.a;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const int item = blockIdx.x / a.kv_heads, head = blockIdx.x - item * a.kv_heads;
    const Part part = find_part(p, item);
    if (!part.any) return;
    const Sequence s = part.s;
    const int block0 = part.block * p.rows, row0 = block0 + wave * 16 * C, rows = s.count * p.group;
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
    uint32_t value[2][kValueWords];
    Place place;
    int page;        // of the tile that is to be requested, -1: none
    bool page_here;  // whether the one that has been requested has one
    constexpr int kKeyTokens = 8 / kKeyUnits;  // tokens whose keys a wave stages at a time
    static_assert(kKeyTokens * kChunks == kWave && kValueUnits == 1, "a wave stages eight tokens");
    const int token8 = 8 * wave;               // the wave's tokens in the tile
    const int key_chunk = lane % kChunks, key_row = lane / kChunks;
    const bool key_column = 8 * key_chunk < a.head_dim;
    const uint32_t key_lane = key_row * p.key_place_bytes + (key_column ? 8 * key_chunk : 0) * kSize;
    const bool value_column = col * kCols < a.head_dim;
    const uint32_t value_lane = 2 * g * p.value_place_bytes + (value_column ? col * kCols : 0) * kSize;
    auto find_place = [&](int t0) { place = place_of(t0 + token8); };
    auto settle = [&]() { page = page_of(place); };
    auto request = [&]() {
        page_here = page >= 0;
        const uint64_t number = (uint32_t)max(page, 0);
        const uint8_t* const k_page = keys + (number * p.key_page_bytes + place.in_page * p.key_place_bytes);
        const uint8_t* const v_page = values + (number * p.value_page_bytes + place.in_page * p.value_place_bytes);
#pragma unroll
        for (int j = 0; j < kKeyUnits; ++j) key[j] = *reinterpret_cast<const KeyPiece*>(k_page + j * kKeyTokens * p.key_place_bytes + key_lane);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint8_t* const from = v_page + t * p.value_place_bytes + value_lane;
            if constexpr (kValueWords == 1) value[t][0] = *reinterpret_cast<const uint32_t*>(from);
            if constexpr (kValueWords == 2) *reinterpret_cast<uint2*>(value[t]) = *reinterpret_cast<const uint2*>(from);
            if constexpr (kValueWords >= 4) {
#pragma unroll
                for (int w = 0; w < kValueWords; w += 4) *reinterpret_cast<uint4*>(value[t] + w) = *reinterpret_cast<const uint4*>(from + 4 * w);
            }
        }
    };
    auto swizzle = [](int step, int group) { return 4 * group + (DP == 64 ? 2 * step : step % 4); };
    auto put = [&](int buffer, int t0) {
        uint8_t* const k_to = tiles[buffer][0];
#pragma unroll
        for (int j = 0; j < kKeyUnits; ++j) {
            const int w = token8 % 32 + j * kKeyTokens + key_row;  // (of 32: rows of two 16-token blocks)
            const int t16 = token8 / 32 * 2 + w / 4 % 2, i = 4 * (w / 8) + w % 4, step = key_chunk / 4, group = key_chunk % 4;
            v4i x;
            if constexpr (FP8) x = v4i{widen2<DT, false>(key[j].x), widen2<DT, true>(key[j].x), widen2<DT, false>(key[j].y), widen2<DT, true>(key[j].y)};
            else x = key[j];
            if (!key_column) x = v4i{0, 0, 0, 0};
            *reinterpret_cast<v4i*>(k_to + ((t16 * kSteps + step) * 64 + group * 16 + (i ^ swizzle(step, group))) * 16) = x;
        }
        uint32_t keep = 0xffffffffu;  // tokens behind the end and without a page are cleared
        if (!page_here || t0 + kSharedTokens > s.length) {
            const int left = page_here ? s.length - (t0 + token8 + 2 * g) : 0;
            keep = (left > 0 ? 0xffffu : 0u) | (left > 1 ? 0xffff0000u : 0u);
        }
        uint8_t* const v_to = tiles[buffer][1] + (token8 / 32 * kCols * 64 + token8 % 32 / 8 * 16 + col) * 16 + g * 4;
        uint32_t pairs[kCols];
#pragma unroll
        for (int f = 0; f < kCols; f += 2) {
            uint32_t even, odd;
            if constexpr (FP8) {
                even = f % 4 == 0 ? widen2<DT, false>(value[0][f / 4]) : widen2<DT, true>(value[0][f / 4]);
                odd = f % 4 == 0 ? widen2<DT, false>(value[1][f / 4]) : widen2<DT, true>(value[1][f / 4]);
            } else {
                even = value[0][f / 2];
                odd = value[1][f / 2];
            }
            pairs[f] = __builtin_amdgcn_perm(odd, even, 0x05040100u) & keep;
            pairs[f + 1] = __builtin_amdgcn_perm(odd, even, 0x07060302u) & keep;
            *reinterpret_cast<uint32_t*>(v_to + f * 1024) = pairs[f];
            *reinterpret_cast<uint32_t*>(v_to + (f + 1) * 1024) = pairs[f + 1];
        }
        bool some = false;
        if (t0 + kSharedTokens > drafted) {
            uint32_t bad = 0;
#pragma unroll
            for (int f = 0; f < kCols; ++f) bad |= unbounded<DT>(pairs[f]);
            some = __any(bad != 0);
        }
        if (lane == 0) {
            exists[buffer][wave] = page_here;
            unsafe[buffer][wave] = some;
        }
    };

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

    Marks<DT, DP, C> marks;
    int end = min(part.to * kTileTokens, s.length);
    if (!a.mask) end = min(end, drafted + (min(block0 + p.rows, rows) - 1) / p.group + 1);
    const int begin = part.from * kTileTokens;
    const int steps = begin < end ? (end - begin + 31) / 32 : 0, tiles_here = (steps + 1) / 2;
    if (steps > 0) {
        find_place(begin);
        settle();
        request();
        find_place(begin + kSharedTokens);
        settle();
        put(0, begin);
        if (tiles_here > 1) request();
        find_place(begin + 2 * kSharedTokens);
    }
    // The queries are here before the loop: waited for within it, a wait would take in the next tile's requests as well.
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int step = 0; step < kSteps; ++step) asm volatile("" : "+v"(query[c][step]));
    if (p.row_info && part.split == 0 && head == 0) {
        for (int r = threadIdx.x; r < p.rows && block0 + r < rows; r += kThreads)
            p.row_info[(long)s.first * p.group + block0 + r] = make_int4(part.slot, part.splits, r, 0);
    }

    const auto load_keys = [&](int i, v4i (&k)[2][kSteps]) {
        const uint8_t* const from = tiles[i >> 1 & 1][0] + (i & 1) * (2 * kSteps * 1024);
#pragma unroll
        for (int step = 0; step < kSteps; ++step)
#pragma unroll
            for (int t = 0; t < 2; ++t) k[t][step] = *reinterpret_cast<const v4i*>(from + key_offset[step % kSwizzles] + (t * kSteps + step) * 1024);
    };
    const auto score_keys = [&](const v4i (&k)[2][kSteps], v4f (&score)[C][2]) {
#pragma unroll
        for (int c = 0; c < C; ++c) score[c][0] = score[c][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int step = 0; step < kSteps; ++step)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int c = 0; c < C; ++c) score[c][t] = mfma16<DT>(k[t][step], query[c][step], score[c][t]);
    };
    constexpr int kAhead = kCols < 8 ? kCols : 8;  // blocks of values read in front of the exponentials: all, up to 128 columns
    v4f score[C][2];
    lds_barrier();
    {
        v4i k[2][kSteps];
        load_keys(0, k);
        score_keys(k, score);
    }
    for (int i = 0; i < steps; ++i) {
        const int buffer = i >> 1 & 1, half = i & 1, h0 = begin + 32 * i, mine = h0 + 8 * g;
        const bool here_page = exists[buffer][4 * half + g] != 0;
        const uint8_t* const v_half = tiles[buffer][1] + half * (kCols * 1024) + lane * 16;
        v4i turned[kAhead];
#pragma unroll
        for (int f = 0; f < kAhead; ++f) turned[f] = *reinterpret_cast<const v4i*>(v_half + f * 1024);
        bool unclean = false;
        if (h0 + 32 > drafted || __any(!here_page || mine + 8 > s.length)) {
            uint32_t seen[C];
            sight<C>(a, s, mine, here_page, seen_to, sees, seen);
#pragma unroll
            for (int c = 0; c < C; ++c) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!(seen[c] >> j & 1)) score[c][j / 4][j % 4] = -INFINITY;
            }
            // Rare: weights of zero do not keep an infinity or a NaN out of the sums.  They are noted for the rows that see their token, and taken out.
            int any = 0;
#pragma unroll
            for (int w = 0; w < kSharedWaves; ++w) any |= unsafe[buffer][w];
            unclean = __builtin_amdgcn_readfirstlane(any) != 0;
            if (unclean) {
                marks.note(seen, reinterpret_cast<const v4i*>(v_half));
#pragma unroll
                for (int f = 0; f < kAhead; ++f) turned[f] = Marks<DT, DP, C>::cleaned(turned[f]);
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
        // The next step's keys: from the second half of a tile on they are in the next one, which all have written by now.  (All have read this one's
        // values too: behind the barrier its buffer is free, but where some blocks are read later.)
        if (half == 1) lds_barrier();
        v4i k[2][kSteps], weight[C];
        v4f score_next[C][2];
        load_keys(i + 1, k);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const float base = top[c] == -INFINITY ? 0.f : top[c];
            float w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = __builtin_amdgcn_exp2f(fmaf(score[c][j / 4][j % 4], scale, -base));
            weight[c] = v4i{pack2<DT>(w[0], w[1]), pack2<DT>(w[2], w[3]), pack2<DT>(w[4], w[5]), pack2<DT>(w[6], w[7])};
        }
        score_keys(k, score_next);
#pragma unroll
        for (int c = 0; c < C; ++c) sum[c] = mfma16<DT>(ones, weight[c], sum[c]);
#pragma unroll
        for (int f = 0; f < kCols; ++f) {
#pragma unroll
            for (int c = 0; c < C; ++c) out[c][f] = mfma16<DT>(turned[f % kAhead], weight[c], out[c][f]);
            if (f + kAhead < kCols) {
                turned[f % kAhead] = *reinterpret_cast<const v4i*>(v_half + (f + kAhead) * 1024);
                if (unclean) turned[f % kAhead] = Marks<DT, DP, C>::cleaned(turned[f % kAhead]);
            }
        }
        if (half == 0) {
            const int next = i / 2 + 1;
            settle();
            if (next < tiles_here) put(next & 1, h0 + kSharedTokens);
            if (next + 1 < tiles_here) request();
            find_place(h0 + 3 * kSharedTokens);
        } else if constexpr (kAhead < kCols) {
            lds_barrier();
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            score[c][0] = score_next[c][0];
            score[c][1] = score_next[c][1];
        }
    }
    marks.apply(out);

    // a lane has DP / 4 neighbouring columns of its rows
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
        if (p.rows == 128) hipLaunchKernelGGL((attention_shared_kernel<DT, FP8, DP, 1>), dim3(grid), dim3(64 * kSharedWaves), 0, stream, p); \
        else if constexpr (DP < 256) hipLaunchKernelGGL((attention_shared_kernel<DT, FP8, DP, 2>), dim3(grid), dim3(64 * kSharedWaves), 0, stream, p); \
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
