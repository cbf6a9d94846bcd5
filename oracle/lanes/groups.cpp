// Beside grouped_gemm.hip and experts.hip on the CPU: the search for a group's tile by itself, and in place of the kernels that run in inline assembly an end.
// Test infrastructure only.
#include <stdio.h>
#include <stdlib.h>

#include "grouped_gemm.h"
#include "skinny_gemm_plan.h"

namespace hfrk {

[[noreturn]] static int not_here(const char* what) {
    fprintf(stderr, "%s does not run on the CPU\n", what);
    abort();
}
bool tiled_size_ok(int, int, int) { not_here("an int8 weight"); }
float make_tiled_plan(int, int, int, int, hfrk_tiled_plan*) { not_here("an int8 weight"); }
size_t tiled_plan_ws_bytes(const hfrk_tiled_plan&, int, int) { not_here("an int8 weight"); }
long tiled_plan_counters(const hfrk_tiled_plan&, int, int) { not_here("an int8 weight"); }
int tiled_launch(const void*, const void*, bool, void*, const void*, int, const float*, int, const float*, int, int, int, int, int, int, const hfrk_tiled_plan&, float*,
                 size_t, int*, hipStream_t, bool) {
    not_here("an int8 weight");
}
int make_rows_plan(int, int, int, hfrk_gemm_plan*) { not_here("an int8 weight"); }
int make_ksplit_plan(int, int, int, hfrk_gemm_plan*) { not_here("an int8 weight"); }
void set_rows_geometry(GemmArgs*, const hfrk_gemm_plan&, bool) { not_here("an int8 weight"); }
int launch_rows_int8_kernel(const GemmArgs&, int, int, int, hipStream_t) { not_here("an int8 weight"); }
int launch_ksplit_int8_kernel(const GemmArgs&, int, int, int, hipStream_t) { not_here("an int8 weight"); }
void turn_k(TiledGemmArgs*, const TiledShape&, bool) { not_here("the tiled kernel"); }
int launch_tiled_grouped_fp8(const TiledGroupedArgs&, int, long, hipStream_t) { not_here("the tiled kernel"); }
int launch_tiled_grouped_int8(const TiledGroupedArgs&, int, long, hipStream_t) { not_here("the tiled kernel"); }

// What find_tile answers to each of `grid` workgroups: five numbers, the expert -1 where it finds none.
static void find_tile_kernel(const GroupedArgs& a, int bm, int32_t (*out)[64][5]) {
    GroupTile t{-1, 0, 0, 0, 0};
    if (!find_tile(a, bm, &t)) t = GroupTile{-1, 0, 0, 0, 0};
    int32_t* const mine = out[blockIdx.x][threadIdx.x];
    mine[0] = t.expert;
    mine[1] = t.first;
    mine[2] = t.rows;
    mine[3] = t.tile;
    mine[4] = t.tiles_m;
}

}  // namespace hfrk

extern "C" {

void lanes_find_tiles(const int32_t* offsets, int experts, int count, int bm, int tiles_n, int grid, int32_t (*out)[64][5]) {
    hfrk::GroupedArgs a{};
    a.offsets = offsets;
    a.experts = experts;
    a.count = count;
    a.tiles_n = tiles_n;
    lanes::launch(dim3(grid), dim3(64), [&] { hfrk::find_tile_kernel(a, bm, out); });
}

long lanes_tiles_bound(int count, int experts, int bm) { return hfrk::grouped_tiles_bound(count, experts, bm); }

}  // extern "C"
