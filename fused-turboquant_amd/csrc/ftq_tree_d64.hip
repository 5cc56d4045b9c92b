// Tree attention at head_dim 64 for the formats of ftq_tree_fast.h.
#include "ftq_tree_fast.h"

namespace ftq {
hipError_t tree_fast_64(const TreeArgs& a, int ct, unsigned grid, hipStream_t st) { return tree_fast_launch<64>(a, ct, grid, st); }
}  // namespace ftq
