// Drafted-token attention, many rows per key: INT8 pools, head_dim 128.
#include "mg_tree_tiles_kernel.cuh"

namespace mg {
template void launch_tree_tiles<false, 128>(const TreeParams&, const TreeGeom&, cudaStream_t);
}  // namespace mg
