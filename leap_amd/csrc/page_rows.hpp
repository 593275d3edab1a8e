// Rows of a sequence between fp32 memory and its pages.
#pragma once

#include "paged_attention.hpp"

namespace leap {

// Rows [row0, row0 + n) of one sequence and layer, [row][kv_head][HD] outside.
// A row is written only into a page of the sequence's own, and read as NaN
// where it has none.  Bound by memory: 8192 rows of 8 heads of 128 in 21 us each
// way (fp32, 134 MB: 6.3 TB/s), 8 bits 19 us in and 27 out (bytes gathered).
struct PageRowsArgs {
    const float *k_in, *v_in;  // (write: either may be NULL)
    float *k_out, *v_out;      // (read)
    void *k, *v;               // the layer's pages
    float *ks, *vs, *bounds;
    const int *table, *refs;   // the sequence's row of the table
    int n_pages, n_kv_heads, rows_log2, row0, n;
};
// 8-bit values: a workgroup turns 16 rows of a KV head to their layout in LDS,
// and writes them 16 bytes a lane; at the range's ends, the range's bytes.
// (8192 rows of 8 KV heads of 128, with the keys: 18.8 us; byte by byte, 50.2)
template <int HD>
__device__ __forceinline__ void page_write_v8(const PageRowsArgs &a)
{
    constexpr int LR = HD / 4, kRows = 256 / LR;  // rows of a pass
    __shared__ alignas(16) int8_t turned[HD][16];
    const int tid = threadIdx.x, c = tid & (LR - 1), end = a.row0 + a.n;
    const int first = a.row0 >> 4, blocks = ((end + 15) >> 4) - first;
    const long long items = (long long)blocks * a.n_kv_heads;
    for (long long i = blockIdx.x; i < items; i += gridDim.x) {
        const int b = (int)(i / a.n_kv_heads), head = (int)(i - (long long)b * a.n_kv_heads), r0 = (first + b) * 16;
        const int page = a.table[r0 >> a.rows_log2];
        if ((unsigned)page >= (unsigned)a.n_pages || a.refs[page] != 1) continue;  // (the same for the workgroup)
        const size_t at = (((size_t)page * a.n_kv_heads + head) << a.rows_log2) + (r0 & ((1 << a.rows_log2) - 1));
        __syncthreads();
#pragma unroll
        for (int r = tid / LR; r < 16; r += kRows) {
            const int row = r0 + r;
            const bool in = row >= a.row0 && row < end;
            const float4 x = in ? reinterpret_cast<const float4 *>(a.v_in)[((long long)(row - a.row0) * a.n_kv_heads + head) * LR + c]
                                : make_float4(0, 0, 0, 0);
            float sc;
            const int q = quantize_row<HD>(x, &sc);
#pragma unroll
            for (int e = 0; e < 4; e++) turned[4 * c + e][r] = (int8_t)(q >> (8 * e));
            if (in && c == 0) a.vs[at + r] = sc;
        }
        __syncthreads();
        int8_t *to = static_cast<int8_t *>(a.v) + at * HD + 16 * tid;
        if (tid < HD) {
            if (r0 >= a.row0 && r0 + 16 <= end) {
                *reinterpret_cast<i32x4 *>(to) = *reinterpret_cast<const i32x4 *>(turned[tid]);
            } else {
                for (int r = max(0, a.row0 - r0); r < min(16, end - r0); r++) to[r] = turned[tid][r];
            }
        }
    }
}
template <int HD, bool Q8>
__global__ __launch_bounds__(256) void page_write_kernel(PageRowsArgs a)
{
    constexpr int LR = HD / 4;
    const float *in = blockIdx.y ? a.v_in : a.k_in;
    if (!in) return;
    if constexpr (Q8)
        if (blockIdx.y) return page_write_v8<HD>(a);
    const long long per_row = (long long)a.n_kv_heads * LR, total = a.n * per_row;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const int r = (int)(i / per_row), w = (int)(i - r * per_row), head = w / LR, c = w & (LR - 1);
        const int row = a.row0 + r, page = a.table[row >> a.rows_log2];
        const float4 x = reinterpret_cast<const float4 *>(in)[i];
        float sc = 0.0f;
        const int q = Q8 ? quantize_row<HD>(x, &sc) : 0;
        if ((unsigned)page >= (unsigned)a.n_pages || a.refs[page] != 1) continue;
        const size_t at = (((size_t)page * a.n_kv_heads + head) << a.rows_log2) + (row & ((1 << a.rows_log2) - 1));
        if constexpr (!Q8) {
            reinterpret_cast<float4 *>(blockIdx.y ? a.v : a.k)[at * LR + c] = x;
        } else {
            reinterpret_cast<int *>(a.k)[at * LR + c] = q;
            if (c == 0) a.ks[at] = sc;
        }
    }
}
template <int HD, bool Q8>
__global__ __launch_bounds__(256) void page_read_kernel(PageRowsArgs a)
{
    constexpr int LR = HD / 4;
    float *out = blockIdx.y ? a.v_out : a.k_out;
    if (!out) return;
    const long long per_row = (long long)a.n_kv_heads * LR, total = a.n * per_row;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const int r = (int)(i / per_row), w = (int)(i - r * per_row), head = w / LR, c = w & (LR - 1);
        const int row = a.row0 + r, page = a.table[row >> a.rows_log2];
        const float nan = __uint_as_float(0x7fc00000u);
        float4 x = make_float4(nan, nan, nan, nan);
        if ((unsigned)page < (unsigned)a.n_pages) {
            const size_t at = (((size_t)page * a.n_kv_heads + head) << a.rows_log2) + (row & ((1 << a.rows_log2) - 1));
            if constexpr (!Q8) {
                x = reinterpret_cast<const float4 *>(blockIdx.y ? a.v : a.k)[at * LR + c];
            } else {
                unsigned q = 0;
                if (!blockIdx.y) {
                    q = (unsigned)reinterpret_cast<const int *>(a.k)[at * LR + c];
                } else {
                    const int8_t *from = static_cast<const int8_t *>(a.v) + (at & ~(size_t)15) * HD + 64 * c + (at & 15);
#pragma unroll
                    for (int e = 0; e < 4; e++) q |= (unsigned)(uint8_t)from[16 * e] << (8 * e);
                }
                x = bytes4((int)q, (blockIdx.y ? a.vs : a.ks)[at]);
            }
        }
        reinterpret_cast<float4 *>(out)[i] = x;
    }
}
// The bounds of the written pages' keys: a wave a page and KV head.
template <int HD, bool Q8>
__global__ __launch_bounds__(256) void page_bounds_kernel(PageRowsArgs a)
{
    const int lane = threadIdx.x & (kWave - 1), R = 1 << a.rows_log2;
    const int first = a.row0 >> a.rows_log2, pages = ((a.row0 + a.n - 1) >> a.rows_log2) - first + 1;
    const int i = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (i >= pages * a.n_kv_heads) return;
    const int j = i / a.n_kv_heads, page = a.table[first + j];
    if ((unsigned)page >= (unsigned)a.n_pages || a.refs[page] != 1) return;
    const size_t head = (size_t)page * a.n_kv_heads + (i - j * a.n_kv_heads), row = head << a.rows_log2;
    page_bounds<HD, Q8>(static_cast<const char *>(a.k) + row * HD * (Q8 ? 1 : 4), Q8 ? a.ks + row : nullptr, a.bounds + head * 2 * HD, R,
                        make_float4(0, 0, 0, 0), false, lane);
}

}  // namespace leap
