// The attention kernels of many rows for heads of 129 to 256 columns.
#include "tree_attention_shared.h"

namespace hfrk {

template int launch_attention_shared<256>(const AttentionArgs& p, int grid, hipStream_t stream);

}  // namespace hfrk
