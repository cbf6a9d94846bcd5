// The attention kernels of many rows for heads of up to 64 columns.
#include "tree_attention_shared.h"

namespace hfrk {

template int launch_attention_shared<64>(const AttentionArgs& p, int grid, hipStream_t stream);

}  // namespace hfrk
