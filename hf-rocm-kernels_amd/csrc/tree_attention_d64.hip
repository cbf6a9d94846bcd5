// The attention kernels for heads of up to 64 columns.
#include "tree_attention_kernel.h"

namespace hfrk {

template int launch_attention<64>(const AttentionArgs& p, int col_blocks, int grid, hipStream_t stream);

}  // namespace hfrk
