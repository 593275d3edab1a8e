// Caches of pages at head_dim 64 (see kernels.hpp).
#include "kernels_paged_table.hpp"

namespace leap_kernels {
template PagedKernels pick_paged_hd<64>(int, bool);
}  // namespace leap_kernels
