// The attention kernels of many rows for heads of 65 to 128 columns.
#include "tree_attention_shared.h"

namespace hfrk {

template int launch_attention_shared<128>(const AttentionArgs& p, int grid, hipStream_t stream);

}  // namespace hfrk
