// Caches of pages at head_dim 128 (see kernels.hpp).
#include "kernels_paged_table.hpp"

namespace leap_kernels {
template PagedKernels pick_paged_hd<128>(int, bool);
}  // namespace leap_kernels
