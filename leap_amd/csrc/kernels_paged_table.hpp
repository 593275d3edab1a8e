// The kernels of caches of pages for one head_dim, included by the
// kernels_paged_*.hip translation units only.
#pragma once

#include "kernels.hpp"

namespace leap_kernels {

template <int HD, int NQ, bool Q8>
PagedKernels paged_table()
{
    return {leap::paged_attention_kernel<HD, NQ, Q8>,
            leap::paged_flat_kernel<HD, NQ, Q8>,
            leap::paged_merge_kernel<HD, Q8>,
            leap::page_write_kernel<HD, Q8>,
            leap::page_read_kernel<HD, Q8>,
            leap::page_bounds_kernel<HD, Q8>,
            leap::page_select_kernel<HD>};
}
template <int HD>
PagedKernels pick_paged_hd(int group, bool q8)
{
    if (q8) return paged_table<HD, 4, true>();
    return group <= 4 ? paged_table<HD, 1, false>() : group == 8 ? paged_table<HD, 2, false>() : paged_table<HD, 4, false>();
}

}  // namespace leap_kernels
