// Drafted-token attention, many rows per key: INT4 pools, head_dim 64.
#include "mg_tree_tiles_kernel.cuh"

namespace mg {
template void launch_tree_tiles<true, 64>(const TreeParams&, const TreeGeom&, cudaStream_t);
}  // namespace mg
