// Prompts, trees and the 8-bit cache at head_dim 64 (see kernels.hpp).
#include "kernels_many_table.hpp"

namespace leap_kernels {
template ManyKernels pick_many_hd<64>(ManyKind, bool);
template RowsKernels pick_rows_hd<64>();
}  // namespace leap_kernels
