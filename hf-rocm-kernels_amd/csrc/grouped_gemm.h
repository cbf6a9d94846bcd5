// Products of rows grouped by expert, and of 8-bit integers: launch arguments, and how a workgroup finds its group.
#pragma once

#include "tiled_gemm.h"

namespace hfrk {

// What the groups are: the same fields for the rows kernel and the tiled one.
struct GroupedArgs {
    const uint8_t* A;
    const uint8_t* B;
    void* D;
    const void* base;  // 16-bit addend or null
    const float* scale_a;
    const float* scale_b;
    const int32_t* offsets;  // group e is rows offsets[e] .. offsets[e+1]; null: one group of all rows
    const int32_t* rows;     // row of A (and of scale_a) for each row of D; null: the same
    int64_t expert_stride;   // bytes from an expert's weight to the next one's
    int64_t sb_expert_stride;
    int base_stride;         // elements between its rows; 0: one row for all (a bias)
    int b_stride, sa_stride, sb_stride;
    int count, a_rows, experts, n, k;
    int d_dtype;
    int vec;                 // rows of D and base take whole 8-byte pieces
    int tiles_n;
};

struct TiledGroupedArgs : TiledGemmArgs {
    const int32_t* offsets;
    const int32_t* rows;
    int64_t expert_stride, sb_expert_stride;
    int count, a_rows, experts;
};

// Tiles of the tiled kernel on groups: the four largest of the dense shapes, and 128 x 128 in five halves of stages, 80 KB, on eight waves that load for themselves, so
// that two workgroups share a compute unit and one multiplies while the other starts or ends.  A group has few tiles and often a short k: start and end are a third
// of the time there (333 tokens on 4 of 60 experts of 2816 x 2048: 128 x 128 79.9 -> 73.8 us, with four waves 75.4; 512 on 8 of 128 of 2048 x 768 77.5 -> 59.1;
// 1024 on 6 of 64 of 2048 x 1408 66.9 -> 58.7).  64 x 128 in the same way gains up to 5 % more where groups have some twenty rows and loses as much above: left out.
// X(index, TM, TN, WM, WN, NST, WGS) as in HFRK_TILED_SHAPES
#define HFRK_GROUP_SHAPES(X) \
    X(0, 4, 2, 2, 4, 5, 1)   \
    X(1, 2, 2, 4, 2, 3, 1)   \
    X(2, 2, 2, 2, 2, 5, 1)   \
    X(3, 2, 1, 2, 2, 3, 2)
#define HFRK_GROUP_PAIRED(X) X(4, 2, 1, 2, 4, 5, 2)

#define HFRK_GROUP_ROW(I, TM, TN, WM, WN, NST, WGS) {32 * TM * WM, 32 * TN * WN, NST, WGS, tiled_half_stages(TM, WM * WN), 64 * (WM * WN + tiled_loader_waves(TM))},
#define HFRK_GROUP_PAIR(I, TM, TN, WM, WN, NST, WGS) {32 * TM * WM, 32 * TN * WN, NST, WGS, true, 64 * WM * WN},
constexpr TiledShape kGroupedShapes[] = {HFRK_GROUP_SHAPES(HFRK_GROUP_ROW) HFRK_GROUP_PAIRED(HFRK_GROUP_PAIR)};
#undef HFRK_GROUP_PAIR
#undef HFRK_GROUP_ROW
constexpr int kGroupedShapeCount = sizeof(kGroupedShapes) / sizeof(kGroupedShapes[0]);

constexpr int kMaxExperts = 512;
constexpr int kOutsideBuffer = 0x7ffffff0;  // beyond the range of every buffer made here

// Inclusive sum over the lanes in front and the lane's own: within rows of 16, then row 0 to row 1 and row 2 to row 3, then the lower half to the upper.
__device__ __forceinline__ int wave_prefix_sum(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
    return x;
}

struct GroupTile {
    int expert, first, rows;  // the group, its first row and its number of rows
    int tile, tiles_m;        // which of the group's tiles_m * tiles_n tiles
};

// The XCDs take workgroups in turn: XCD x gets one contiguous range of `total` ids, so that neighbours share an L2.  -1: none is left.
__device__ __forceinline__ int xcd_range_id(int block, int total) {
    const int x = block & (kNumXCD - 1), slot = block / kNumXCD, per = total / kNumXCD, extra = total % kNumXCD;
    return slot < per + (x < extra ? 1 : 0) ? x * per + min(x, extra) + slot : -1;
}

// Which tile of which group this workgroup has: tiles of `bm` rows, all groups' tiles in the order of the experts.  Group sizes are known on the
// device only, so a launch has a workgroup for every tile there can be (grouped_tiles_bound) and those behind the last one find none.  Each
// wave looks for itself, a lane at up to EPL experts.  Offsets that do not increase, or pass the rows, cannot lead outside: each is cut to 0 .. count, and a tile is one of a
// group's own or none.
template <int EPL, typename Args>
__device__ __forceinline__ bool find_tile_of(const Args& a, int bm, GroupTile* t) {
    const int lane = threadIdx.x & 63;
    int edge[EPL + 1], tiles[EPL];
#pragma unroll
    for (int j = 0; j <= EPL; ++j) {
        const int e = min(lane * EPL + j, a.experts);
        edge[j] = a.offsets[e];
    }
    int mine = 0;
#pragma unroll
    for (int j = 0; j <= EPL; ++j) edge[j] = min(max(edge[j], 0), a.count);
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
        tiles[j] = edge[j + 1] > edge[j] ? (edge[j + 1] - edge[j] + bm - 1) / bm : 0;
        mine += tiles[j];
    }
    const int upto = wave_prefix_sum(mine);
    const int total = __builtin_amdgcn_readlane(upto, 63) * a.tiles_n;
    const int id = xcd_range_id(blockIdx.x, total);
    if (id < 0) return false;
    const uint64_t behind = __ballot(upto * a.tiles_n > id);
    if (behind == 0) return false;
    const int owner = __builtin_ctzll(behind);
    int left = id - __builtin_amdgcn_readlane(upto - mine, owner) * a.tiles_n;
    bool found = false;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
        const int tm = __builtin_amdgcn_readlane(tiles[j], owner);
        if (!found && left >= 0 && left < tm * a.tiles_n) {
            found = true;
            t->expert = owner * EPL + j;
            t->first = __builtin_amdgcn_readlane(edge[j], owner);
            t->rows = __builtin_amdgcn_readlane(edge[j + 1], owner) - t->first;
            t->tile = left;
            t->tiles_m = tm;
        }
        left -= found ? 0 : tm * a.tiles_n;
    }
    return found;
}

template <typename Args>
__device__ __forceinline__ bool find_tile(const Args& a, int bm, GroupTile* t) {
    if (!a.offsets) {
        t->expert = 0;
        t->first = 0;
        t->rows = a.count;
        t->tiles_m = (a.count + bm - 1) / bm;
        t->tile = xcd_range_id(blockIdx.x, t->tiles_m * a.tiles_n);
        return t->tile >= 0;
    }
    if (a.experts <= 64) return find_tile_of<1>(a, bm, t);
    return a.experts <= 128 ? find_tile_of<2>(a, bm, t) : find_tile_of<kMaxExperts / 64>(a, bm, t);
}

// The most tiles of `bm` rows that groups of `count` rows together can have: every group's last one may be partly filled.
inline long grouped_tiles_bound(int count, int experts, int bm) { return (long)count / bm + (experts < count ? experts : count); }

// tiled_grouped_fp8.hip, tiled_grouped_int8.hip, tiled_int8.hip: the tiled kernel on groups and on one int8 weight.
int launch_tiled_grouped_fp8(const TiledGroupedArgs& args, int shape, long grid, hipStream_t stream);
int launch_tiled_grouped_int8(const TiledGroupedArgs& args, int shape, long grid, hipStream_t stream);
int launch_tiled_int8(const TiledGemmArgs& args, int shape, hipStream_t stream);

}  // namespace hfrk
