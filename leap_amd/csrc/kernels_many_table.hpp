// The kernels of prompts, trees and the 8-bit cache for one head_dim, included
// by the kernels_many_*.hip translation units only.
#pragma once

#include "kernels.hpp"

namespace leap_kernels {

template <int HD>
ManyKernels pick_many_hd(int nb, bool q8)
{
    const ManyFn append = q8 ? leap::many_append_kernel<HD, true> : leap::many_append_kernel<HD, false>;
#define LEAP_CASE(NB) \
    if (nb == NB) return {append, q8 ? leap::many_attention_kernel<HD, NB, true> : leap::many_attention_kernel<HD, NB, false>};
    LEAP_CASE(1) LEAP_CASE(2) LEAP_CASE(4)
#undef LEAP_CASE
    return {nullptr, nullptr};
}

template <int HD>
RowsKernels pick_rows_hd()
{
    return {leap::q8_write_kernel<HD>, leap::q8_read_kernel<HD>};
}

}  // namespace leap_kernels
