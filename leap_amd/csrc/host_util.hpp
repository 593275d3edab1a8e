// What the library's host sides share.
#pragma once

#include <hip/hip_runtime.h>

#include <string>

namespace leap_host {

template <typename T>
struct same_type {
    using type = T;
};

// Enqueue fn<<<grid, block, 0, stream>>>(args...) and return that launch's
// own status (not the thread's sticky last error, which may be older).
template <typename... P>
hipError_t launch_k(void (*fn)(P...), dim3 grid, dim3 block, hipStream_t stream, typename same_type<P>::type... args)
{
    void *kargs[] = {static_cast<void *>(&args)...};
    return hipLaunchKernel(reinterpret_cast<const void *>(fn), grid, block, kargs, 0, stream);
}

// Whether `device` (the current one) places workgroups whose ids are equal
// modulo 8 on one XCD, as the merges need: 0, or a negative errno value and
// why.  Checked on a launch of n_wg workgroups.
int check_placement(int device, int n_wg, std::string *why);

}  // namespace leap_host
