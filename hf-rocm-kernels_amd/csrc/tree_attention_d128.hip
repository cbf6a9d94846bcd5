// The attention kernels for heads of 65 to 128 columns.
#include "tree_attention_kernel.h"

namespace hfrk {

template int launch_attention<128>(const AttentionArgs& p, int col_blocks, int grid, hipStream_t stream);

}  // namespace hfrk
