// The attention kernels for heads of 129 to 256 columns.
#include "tree_attention_kernel.h"

namespace hfrk {

template int launch_attention<256>(const AttentionArgs& p, int col_blocks, int grid, hipStream_t stream);

}  // namespace hfrk
