// Tree attention at head_dim 256 for the formats of ftq_tree_fast.h.
#include "ftq_tree_fast.h"

namespace ftq {
hipError_t tree_fast_256(const TreeArgs& a, int ct, unsigned grid, hipStream_t st) { return tree_fast_launch<256>(a, ct, grid, st); }
}  // namespace ftq
