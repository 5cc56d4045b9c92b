// Tree attention at head_dim 128 for the formats of ftq_tree_fast.h.
#include "ftq_tree_fast.h"

namespace ftq {
hipError_t tree_fast_128(const TreeArgs& a, int ct, unsigned grid, hipStream_t st) { return tree_fast_launch<128>(a, ct, grid, st); }
}  // namespace ftq
