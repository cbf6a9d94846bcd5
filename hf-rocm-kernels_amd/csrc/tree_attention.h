// Shared by the attention kernels and their launcher: the arguments, and which part of the work a workgroup has.
#pragma once

#include "hfrk_internal.h"

namespace hfrk {

constexpr int kWaveTokens = 32;  // cached tokens a wave takes at a time
constexpr int kDirectWaves = 4;  // of a workgroup that holds keys and values in registers

struct AttentionArgs {
    hfrk_attention_args a;
    float log2_scale;         // softmax scale * log2(e)
    int group;                // query heads per key head
    int rows;                 // rows of a block: C * 16, each a (token, head of the group)
    int tile;                 // cached tokens that work is dealt out in
    int work;                 // workgroups the card has room for at once
    int shares;               // into how many workgroups one's share may be cut
    int slots;                // partial results the workspace holds, per key head
    uint32_t page_magic;      // (t / 8) / (page_size / 8) as a multiplication: n * magic >> (32 + page_shift), or n >> page_shift where magic is 0
    int page_shift;
    uint32_t key_page_bytes, key_place_bytes, value_page_bytes, value_place_bytes;  // strides, where 32 bits hold them (`narrow`)
    float* partial;           // [slots * kv_heads][rows][head_dim], divided by nothing
    float2* partial_ml;       // [slots * kv_heads][rows]: the scale that weights were made with (in log2 units) and their sum
    int4* row_info;           // [tokens * group]: first slot, splits, row in its block
    long join_first;          // the first (row, key head) of a join's launch
};

// A sequence's drafted tokens (rows first .. first + count of the query), its cached ones (these included) as far as its row of the page table
// reaches, and the place of the first drafted one: what is in front of it is seen by all.
struct Sequence {
    int first, count, length, drafted;
};

__device__ __forceinline__ Sequence sequence(const AttentionArgs& p, int b) {
    Sequence s;
    if (p.a.starts) {
        s.first = min(max(p.a.starts[b], 0), p.a.tokens);
        s.count = min(max(p.a.starts[b + 1], s.first), p.a.tokens) - s.first;
    } else {
        s.count = p.a.tokens / p.a.seqs;
        s.first = b * s.count;
    }
    const long room = (long)p.a.table_columns * p.a.page_size;
    const int length = max(p.a.lengths[b], 0);
    s.length = length < room ? length : (int)room;
    s.drafted = length - s.count;
    return s;
}

// What a workgroup does: row block `block` of sequence `b`, cached tokens [from, to).
struct Part {
    int b, block, split, splits, slot;   // slot: where its partial result goes (splits > 1)
    int from, to;                        // its tokens; from >= to: none
    Sequence s;
    bool any;
};

// Inclusive sum over the wave's lanes: within rows of 16 by shifts of 1, 2, 4, 8, then the first and third row's last lane to the rows behind them, then the
// first half's to the second half.  (By exchanges through LDS a workgroup's start took 0.5 us longer.)
__device__ __forceinline__ int lane_prefix(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
}

__device__ __forceinline__ uint32_t lanes_sum(uint32_t v) {  // over the wave; as wave_sum
    const auto halves = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = halves[0] + halves[1];
    const auto rows = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = rows[0] + rows[1];
    v += __builtin_amdgcn_update_dpp(0u, v, 0x128, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0u, v, 0x124, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0u, v, 0x122, 0xf, 0xf, true);
    return v + __builtin_amdgcn_update_dpp(0u, v, 0x121, 0xf, 0xf, true);
}

// The list of work: for every sequence row blocks x splits of its tiles.  How many tiles a workgroup takes follows from all sequences' lengths as they
// are now (in a captured graph too), so that a long one does not keep a few workgroups busy while the others are done.  Each wave makes the list by
// itself: lanes are sequences.
//
// Of the whole's share of a workgroup, a half and so on of it (p.shares), and of what lets all workgroups run at once, that is taken which ends
// first: where all run at once, with the longest; else with the whole's share and half a workgroup more.  A workgroup costs about two tiles by itself.
// (64 lengths from 1 to 8192 in fp8: all at once 131 us, the share 101, half of it 97, a quarter 110.)
__device__ __forceinline__ Part find_part(const AttentionArgs& p, int item) {
    const int lane = threadIdx.x & (kWave - 1);
    Part part = {};
    struct Amount {
        int blocks, tiles;
        Sequence s;
    };
    auto look = [&](int b) {
        Amount m = {};
        if (b < p.a.seqs) {
            m.s = sequence(p, b);
            m.blocks = (int)((uint32_t)(m.s.count * p.group + p.rows - 1) / (uint32_t)p.rows);
            m.tiles = (int)((uint32_t)(m.s.length + p.tile - 1) / (uint32_t)p.tile);
        }
        return m;
    };
    const Amount first = look(lane);  // the first 64 sequences stay in registers, mostly all
    auto amount = [&](int b0) { return b0 == 0 ? first : look(b0 + lane); };
    // ceil(tiles / chunk); the half keeps the quotient's rounding from an integer for tiles + chunk below 2^21
    auto splits_of = [](int tiles, int chunk) { return max(1, (int)(((float)(tiles + chunk) - 0.5f) * __builtin_amdgcn_rcpf((float)chunk))); };
    uint32_t total = 0, least_items = 0;  // (the host has bounded blocks * tiles)
    for (int b0 = 0; b0 < p.a.seqs; b0 += kWave) {
        const Amount m = amount(b0);
        total += lanes_sum((uint32_t)(m.blocks * m.tiles));
        least_items += lanes_sum((uint32_t)m.blocks);
    }
    auto items_of = [&](int chunk) {
        uint32_t items = 0;
        for (int b0 = 0; b0 < p.a.seqs; b0 += kWave) {
            const Amount m = amount(b0);
            items += lanes_sum((uint32_t)(m.blocks * splits_of(m.tiles, chunk)));
        }
        return items;
    };
    const uint32_t room = (uint32_t)max(1, p.work / p.a.kv_heads);
    int chunk = max(1, (int)((total + room - 1) / room));
    if (p.shares > 1 && least_items > 0) {
        const int share = chunk;
        float best = 3e38f;
        uint32_t at_once = 0;
        for (int k = 1; k <= p.shares + 1; ++k) {
            const int now = k <= p.shares ? (share + k - 1) / k : (int)((uint64_t)share * at_once / room) + 1;
            if (k > p.shares && (at_once <= room || least_items > room)) break;
            const uint32_t items = items_of(now);
            if (k == 1) at_once = items;
            const float ends = items <= room ? (float)now : ((float)total + 2.f * (float)items) * __builtin_amdgcn_rcpf((float)room) + 0.5f * (float)now;
            if (ends < best) {
                best = ends;
                chunk = now;
            }
        }
    }
    chunk = __builtin_amdgcn_readfirstlane(chunk);
    int items = 0, slots = 0;
    for (int b0 = 0; b0 < p.a.seqs; b0 += kWave) {
        const Amount m = amount(b0);
        const Sequence s = m.s;
        const int splits = splits_of(m.tiles, chunk);
        const int n = m.blocks * splits, held = splits > 1 ? n : 0;
        const int items_to = items + lane_prefix(n), slots_to = slots + lane_prefix(held);
        const uint64_t found = __ballot(n > 0 && item >= items_to - n && item < items_to);
        if (found) {
            const int who = __ffsll((unsigned long long)found) - 1;
            const auto of = [who](int v) { return __builtin_amdgcn_readlane(v, who); };  // (into scalar registers: the same for the whole workgroup)
            const int at = item - (of(items_to) - of(n)), all = of(m.tiles);
            part.b = b0 + who;
            part.splits = of(splits);
            part.block = (uint32_t)at / (uint32_t)part.splits;
            part.split = at - part.block * part.splits;
            part.slot = of(slots_to) - of(held) + at;
            const int even = (int)((uint32_t)(all + part.splits - 1) / (uint32_t)part.splits);
            part.from = part.split * even * p.tile;
            part.to = min((part.split + 1) * even, all) * p.tile;
            part.s = {of(s.first), of(s.count), of(s.length), of(s.drafted)};
            // The workspace has room for every list of starts that do not decrease; with others the sums may wrap, and what has no room is left out.
            const int slot0 = part.slot - part.split;
            part.any = part.splits == 1 || (slot0 >= 0 && part.splits <= p.slots - slot0);
            return part;
        }
        items = __builtin_amdgcn_readlane(items_to, kWave - 1);
        slots = __builtin_amdgcn_readlane(slots_to, kWave - 1);
    }
    return part;
}

// Rows are dealt to lanes by C blocks of 16; one file per padded head size instantiates them.
template <int DP>
int launch_attention(const AttentionArgs& p, int col_blocks, int grid, hipStream_t stream);

// The same for many rows, which share keys and values in LDS (tree_attention_shared.h): 128 or (up to 128 columns) 256 rows a block.
template <int DP>
int launch_attention_shared(const AttentionArgs& p, int grid, hipStream_t stream);

}  // namespace hfrk
