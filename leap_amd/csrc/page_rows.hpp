// Rows of a sequence between fp32 memory and its pages.
#pragma once

#include "paged_attention.hpp"

namespace leap {

// Rows [row0, row0 + n) of one sequence and layer, [row][kv_head][HD] outside.
// A row is written only into a page of the sequence's own, and read as NaN
// where it has none.
struct PageRowsArgs {
    const float *k_in, *v_in;  // (write: either may be NULL)
    float *k_out, *v_out;      // (read)
    void *k, *v;               // the layer's pages
    float *ks, *vs, *bounds;
    const int *table, *refs;   // the sequence's row of the table
    int n_pages, n_kv_heads, rows_log2, row0, n;
};
template <int HD, bool Q8>
__global__ __launch_bounds__(256) void page_write_kernel(PageRowsArgs a)
{
    constexpr int LR = HD / 4;
    const float *in = blockIdx.y ? a.v_in : a.k_in;
    if (!in) return;
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
            if (!blockIdx.y) {
                reinterpret_cast<int *>(a.k)[at * LR + c] = q;
            } else {
                int8_t *to = static_cast<int8_t *>(a.v) + (at & ~(size_t)15) * HD + 64 * c + (at & 15);
#pragma unroll
                for (int e = 0; e < 4; e++) to[16 * e] = (int8_t)(q >> (8 * e));
            }
            if (c == 0) (blockIdx.y ? a.vs : a.ks)[at] = sc;
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
