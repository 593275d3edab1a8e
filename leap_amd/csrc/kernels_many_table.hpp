// The kernels of prompts, trees and the 8-bit cache for one head_dim, included
// by the kernels_many_*.hip translation units only.
#pragma once

#include "kernels.hpp"
#include "wide_attention.hpp"

namespace leap_kernels {

template <int HD>
ManyKernels pick_many_hd(int nb, bool q8)
{
    const ManyFn append = q8 ? leap::many_append_kernel<HD, true> : leap::many_append_kernel<HD, false>;
    if (nb == 1)
        return q8 ? ManyKernels{append, leap::many_attention_kernel<HD, 1, 8, true>, leap::many_merge_kernel<HD, 16>, 8, 16}
                  : ManyKernels{append, leap::many_attention_kernel<HD, 1, 4, false>, leap::many_merge_kernel<HD, 16>, 4, 16};
    return {append, q8 ? leap::wide_attention_kernel<HD, true> : leap::wide_attention_kernel<HD, false>,
            leap::many_merge_kernel<HD, leap::kWideRows>, leap::kWideWaves, leap::kWideRows};
}

template <int HD>
RowsKernels pick_rows_hd()
{
    return {leap::q8_write_kernel<HD>, leap::q8_read_kernel<HD>};
}

}  // namespace leap_kernels
