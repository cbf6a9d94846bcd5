// Tiled GEMM on rows grouped by expert, fp8 codes (tiled_gemm_kernel.h).
#include "tiled_gemm_kernel.h"

namespace hfrk {

int launch_tiled_grouped_fp8(const TiledGroupedArgs& args, int shape, long grid, hipStream_t stream) {
    return launch_tiled_groups<false>(args, shape, grid, stream);
}

}  // namespace hfrk
