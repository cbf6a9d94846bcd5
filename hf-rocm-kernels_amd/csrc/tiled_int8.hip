// Tiled GEMM on int8 codes (tiled_gemm_kernel.h): v_mfma_i32_32x32x32_i8 at the rate of the fp8 instruction, everything else alike.
#include "tiled_gemm_kernel.h"

namespace hfrk {

int launch_tiled_int8(const TiledGemmArgs& args, int shape, hipStream_t stream) { return launch_tiled<false, true>(args, shape, stream); }

}  // namespace hfrk
