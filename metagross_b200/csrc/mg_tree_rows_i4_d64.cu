// Drafted-token attention, few rows per key: INT4 pools, head_dim 64.
#include "mg_tree_rows_kernel.cuh"

namespace mg {
template void launch_tree_rows<true, 64>(const TreeParams&, const TreeGeom&, cudaStream_t);
}  // namespace mg
