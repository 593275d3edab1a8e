// The kernels of caches of pages for one head_dim, included by the
// kernels_paged_*.hip translation units only.
#pragma once

#include "kernels.hpp"

namespace leap_kernels {

template <int HD, bool Q8>
PagedKernels paged_table()
{
    return {{leap::paged_attention_kernel<HD, 4, Q8>, leap::paged_attention_kernel<HD, 8, Q8>},
            leap::paged_merge_kernel<HD, Q8>,
            leap::page_write_kernel<HD, Q8>,
            leap::page_read_kernel<HD, Q8>,
            leap::page_bounds_kernel<HD, Q8>,
            leap::page_select_kernel<HD>};
}
template <int HD>
PagedKernels pick_paged_hd(bool q8)
{
    return q8 ? paged_table<HD, true>() : paged_table<HD, false>();
}

}  // namespace leap_kernels
