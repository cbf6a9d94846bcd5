// Shared by the attention kernels and their launcher: the arguments, and which part of the work a workgroup has.
#pragma once

#include "hfrk_internal.h"

namespace hfrk {

constexpr int kAttentionThreads = 256;
constexpr int kAttentionWaves = kAttentionThreads / kWave;
constexpr int kWaveTokens = 32;                                   // cached tokens a wave takes at a time
constexpr int kTileTokens = kWaveTokens * kAttentionWaves;        // and a workgroup

struct AttentionArgs {
    hfrk_attention_args a;
    float log2_scale;         // softmax scale * log2(e)
    int group;                // query heads per key head
    int rows;                 // rows of a block: C * 16, each a (token, head of the group)
    int work;                 // tiles per workgroup are chosen so that about this many have some
    int slots;                // partial results the workspace holds, per key head
    uint32_t page_magic;      // (t / 8) / (page_size / 8) as a multiplication: n * magic >> (32 + page_shift), or n >> page_shift where magic is 0
    int page_shift;
    uint32_t key_page_bytes, key_place_bytes, value_page_bytes, value_place_bytes;  // strides, where 32 bits hold them (`narrow`)
    float* partial;           // [slots * kv_heads][rows][head_dim], divided by nothing
    float2* partial_ml;       // [slots * kv_heads][rows]: largest score (in log2 units) and sum
    int4* row_info;           // [tokens * group]: first slot, splits, row in its block
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
    int from, to;                        // in tiles of kTileTokens
    Sequence s;
    bool any;
};

template <typename T>
__device__ __forceinline__ T lane_prefix(T v, int lane) {  // inclusive sum over the wave's lanes
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const T below = __shfl_up(v, d);
        if (lane >= d) v += below;
    }
    return v;
}

// The list of work: for every sequence row blocks x splits of its tiles.  The tiles a workgroup takes follow from all sequences' lengths as they are
// now (in a captured graph too), so that a long one does not keep a few workgroups busy while the others are done.  Each wave makes the list by
// itself: lanes are sequences.
__device__ __forceinline__ Part find_part(const AttentionArgs& p, int item) {
    const int lane = threadIdx.x & (kWave - 1);
    Part part = {};
    auto amount = [&](int b, int& blocks, int& tiles) {
        blocks = tiles = 0;
        Sequence s = {0, 0, 0, 0};
        if (b < p.a.seqs) {
            s = sequence(p, b);
            blocks = (int)(((long)s.count * p.group + p.rows - 1) / p.rows);
            tiles = (s.length + kTileTokens - 1) / kTileTokens;
        }
        return s;
    };
    long total = 0;
    for (int b0 = 0; b0 < p.a.seqs; b0 += kWave) {
        int blocks, tiles;
        amount(b0 + lane, blocks, tiles);
        long mine = (long)blocks * tiles;
        if (p.a.seqs > 1) {
#pragma unroll
            for (int d = 1; d < kWave; d <<= 1) mine += __shfl_xor(mine, d);
            total += mine;
        } else {
            total = __shfl(mine, 0);
        }
    }
    const long share = (total * p.a.kv_heads + p.work - 1) / p.work;
    const int chunk = __builtin_amdgcn_readfirstlane(share < 1 ? 1 : (int)share);
    int items = 0, slots = 0;
    for (int b0 = 0; b0 < p.a.seqs; b0 += kWave) {
        int blocks, tiles;
        const Sequence s = amount(b0 + lane, blocks, tiles);
        const int splits = max(1, (tiles + chunk - 1) / chunk);
        const int n = blocks * splits, held = splits > 1 ? n : 0;
        const int items_to = items + (p.a.seqs > 1 ? lane_prefix(n, lane) : n);
        const int slots_to = slots + (p.a.seqs > 1 ? lane_prefix(held, lane) : held);
        const uint64_t found = __ballot(n > 0 && item >= items_to - n && item < items_to);
        if (found) {
            const int who = __ffsll((unsigned long long)found) - 1;
            const auto of = [who](int v) { return __builtin_amdgcn_readlane(v, who); };  // (into scalar registers: the same for the whole workgroup)
            const int at = item - (of(items_to) - of(n));
            part.b = b0 + who;
            part.splits = of(splits);
            part.block = (uint32_t)at / (uint32_t)part.splits;
            part.split = at - part.block * part.splits;
            part.slot = of(slots_to) - of(held) + at;
            part.from = part.split * chunk;
            part.to = min(part.from + chunk, of(tiles));
            part.s = {of(s.first), of(s.count), of(s.length), of(s.drafted)};
            part.any = true;
            return part;
        }
        items = __builtin_amdgcn_readlane(items_to, p.a.seqs > 1 ? kWave - 1 : 0);
        slots = __builtin_amdgcn_readlane(slots_to, p.a.seqs > 1 ? kWave - 1 : 0);
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
