// Prompts, trees and the 8-bit cache at head_dim 128, and the moves of
// tree_keep (see kernels.hpp).
#include "kernels_many_table.hpp"

namespace leap_kernels {
template ManyKernels pick_many_hd<128>(ManyKind, bool);
template RowsKernels pick_rows_hd<128>();
KeepFn pick_keep(bool q8) { return q8 ? leap::tree_keep_kernel<true> : leap::tree_keep_kernel<false>; }
}  // namespace leap_kernels
