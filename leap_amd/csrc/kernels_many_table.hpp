// The kernels of prompts, trees and the 8-bit cache for one head_dim, included
// by the kernels_many_*.hip translation units only.
#pragma once

#include "kernels.hpp"
#include "wide_attention.hpp"

namespace leap_kernels {

template <int HD>
ManyKernels pick_many_hd(ManyKind kind, bool q8)
{
    constexpr int R = leap::kManyRows, B = leap::kWideRows;
    const ManyFn append = q8 ? leap::many_append_kernel<HD, true> : leap::many_append_kernel<HD, false>;
    if (kind == kManyWide)
        return {append, q8 ? leap::wide_attention_kernel<HD, true> : leap::wide_attention_kernel<HD, false>,
                {leap::many_merge_kernel<HD, B, 4>, leap::many_merge_kernel<HD, B, 16>}, leap::kWideWaves, B};
    // (tiles of 16 rows are spread in groups of fewer than 8: never the merge of many)
    const ManyFn merge = leap::many_merge_kernel<HD, R, 4>;
    if (!q8) return {append, leap::many_attention_kernel<HD, 4, false, false>, {merge, nullptr}, 4, R};
    return {append, kind == kManyStep ? leap::many_attention_kernel<HD, 8, true, true> : leap::many_attention_kernel<HD, 8, true, false>,
            {merge, nullptr}, 8, R};
}

template <int HD>
RowsKernels pick_rows_hd()
{
    return {leap::q8_write_kernel<HD>, leap::q8_read_kernel<HD>};
}

}  // namespace leap_kernels
