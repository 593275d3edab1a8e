// Attention of one new token of each sequence over a cache kept in pages, of
// fp32 or of 8-bit values.
//
// A page holds R rows (16, 32, 64 or 128) of every KV head of one layer; a
// sequence's pages are named by its row of a table.  Per layer the arrays are
//   fp32    k, v    [page][kv_head][R][HD]
//   8 bits  k8      [page][kv_head][R][HD]
//           v8      [page][kv_head][R / 16][HD][16]  (16 rows, dim by dim)
//           ks, vs  [page][kv_head][R]
// so that a KV head's rows of a page lie together, and the operands of both
// products are read from memory as the matrix instructions take them.
//
// A workgroup takes one (sequence, KV head) and one run of tiles of positions;
// its waves take tiles in turn, each with an online softmax of its own, and
// their results are combined in LDS.  The runs of one group leave records
// (output, log2 of the sum) that the last one to arrive adds up, or, where a
// group's runs are spread over the XCDs, a second launch.  A launch attends
// either to all pages of a sequence or to a list of them for each KV head
// (ascending, the new row's page last): the rows are then numbered along the
// list, and only the last page may be partly filled, as without a list.
//
// Bound by memory in batches: 16 sequences of 411 to 7300 rows, 64/8 heads of
// 128, 675 MB in 108 us (6.2 TB/s), 16 of 8192, 32/8 heads, in 160 us (6.7);
// 8 bits, 32 of 8192, 555 MB in 100 us (5.5).  Small steps are bound by
// latency: one sequence of 4096 11.6 us, of 256 rows with 4 KV heads of 64 6.9
// (page numbers, rows, a tile, records).  Four waves a workgroup and one or two
// workgroups a CU: more, shorter runs stream less (8 tiles each 200 us for 160).
//
// Products, m = lane % 16, g = lane / 16.
//   fp32: v_mfma_f32_4x4x1_16b_f32, 4 q heads (a quad) by 4 rows and blocks of
//     16: a lane's K is row m of 16, dims 16 f + 4 g.., and after the sum over
//     the four g it has the score of head g of the quad at position m: every
//     lane one, whatever the scores' number.  A V load is whole rows, 4 dims a
//     lane, whose weights of the quad come through LDS.  16x16x4 products,
//     which have no use for 12 of 16 columns with 4 heads, take four times as
//     long (eight tiles a CU at once: 1.9 us for 0.5).
//   8 bits: v_mfma_i32_16x16x64_i8 on the cache's bytes as they are.  S^T = K
//     Q^T: a lane holds K's row m and q head m, and gets the scores of 4
//     positions for head m; O^T = V^T P^T takes those registers as its B
//     operand.  The other operand, q or the probabilities times the value
//     rows' scales, is a 30-bit fixed-point number over a power of two just
//     above the largest of its head row (q) or of its tile (probabilities), as
//     four signed digits of 8 bits; the four integer sums are exact and are put
//     together in fp32.  What is lost is 2^-30 of that largest element.  O is
//     held in units of a power of two of the weighted values' size.
#pragma once

#include "many_attention.hpp"

namespace leap {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kPagedWaves = 4;       // waves of a workgroup
constexpr int kPagedSplits = 64;     // runs of a group, at most: a lane each in the merge
constexpr int kPagedHeads = 16;      // q heads of a KV head, at most
// Probabilities are 2^(score - reference - bias), and the reference moves when
// a score exceeds it by more than kPagedMargin.  fp32: with a bias of 20 sums
// of up to 2^16 probabilities stay below 1, and weighted values below the
// largest value.  8 bits: probabilities are at most 1, and the weighted values
// are in units of a power of two of their size, O's unit, which moves up with
// them and down where the reference leaves them behind (without one, values
// below 1e-21 lost bits: 0.1% at 1e-25).  It costs 0.1 to 0.2 us of small steps
// and nothing of large ones.
constexpr float kPagedMargin = 4.0f;
template <bool Q8>
constexpr float kPagedBias = Q8 ? kPagedMargin : 20.0f;

// One launch over one layer.
struct PagedArgs {
    const float *q, *k_new, *v_new;  // rows of [n_heads*HD], [n_kv_heads*HD]
    float *out;
    void *k, *v;                     // the layer's pages
    float *ks, *vs;                  // 8 bits: their scales
    float *bounds;                   // the layer's [page][kv_head][2][HD], or NULL
    const float4 *rope;
    const int *pos;
    const int *table;                // [sequence][width]
    const int *refs;                 // [page]
    const int *whole;                // [sequence]: its pages ahead of the first that is missing
    const int *lists;                // [group][keep] pages (keep 0: none, all pages of the table)
    float *ws_o, *ws_lse;            // records: [group][split][q head][HD], [group][split][q head]
    int *counters;                   // [group], kCtrStride apart, zero between launches
    int width, keep, n_pages;
    int n_seq, max_pos, n_heads, n_kv_heads, group;
    int rows_log2;                   // R = 1 << rows_log2
    int chunk, splits;               // tiles of a run, runs of the longest group (flat: most groups of an XCD)
    int blocks;                      // blocks of 16 rows of the longest group
    int spread;                      // a group's runs lie on all XCDs, and paged_merge_kernel adds up their records
    float scale_log2;
    FastDiv by_kv_heads, by_splits, by_chunk, by_groups;
};

// A word that the kernel does not write, at an address that is the same in all
// lanes: by way of the scalar cache, so that the wait for it is not one for
// the rows that are on their way.
__device__ __forceinline__ int uniform_load(const int *p)
{
    typedef __attribute__((address_space(4))) const int ConstInt;
    return *(ConstInt *)(uintptr_t)p;
}

// What a group (sequence, KV head) attends to.
struct PagedPlace {
    int seq, kvh, pos;
    const int *list;     // page numbers
    int n_list, rows;    // pages, and rows along the list with the new one
    bool skip;           // a position out of range, or a page of its rows missing
};
__device__ __forceinline__ PagedPlace paged_place(const PagedArgs &a, int gi)
{
    PagedPlace p;
    p.seq = (int)fast_div((uint32_t)gi, a.by_kv_heads);
    p.kvh = gi - p.seq * a.n_kv_heads;
    p.list = a.keep ? a.lists + (size_t)gi * a.keep : a.table + (size_t)p.seq * a.width;
    return p;
}
// (its position known, and how many of its pages are there)
__device__ __forceinline__ void paged_rows(const PagedArgs &a, PagedPlace &p, int whole)
{
    const int at = p.pos >> a.rows_log2;
    p.n_list = a.keep ? min(a.keep, at + 1) : at + 1;
    p.rows = ((p.n_list - 1) << a.rows_log2) + (p.pos & ((1 << a.rows_log2) - 1)) + 1;
    p.skip = p.pos < 0 || p.pos > a.max_pos || at >= whole;
}
// NaN into a skipped sequence's output row, by `step` threads.
template <int HD>
__device__ __forceinline__ void paged_skip(const PagedArgs &a, const PagedPlace &p, int i0, int step = kPagedWaves * kWave)
{
    fill_nan<HD>(a.out, ((size_t)p.seq * a.n_heads + p.kvh * a.group) * (HD / 4), a.group * (HD / 4), i0, step);
}
// The runs of a group of so many tiles (run i: tiles [i chunk, (i + 1) chunk)).
__device__ __forceinline__ int paged_runs(const PagedArgs &a, int tiles) { return (int)fast_div((uint32_t)(tiles + a.chunk - 1), a.by_chunk); }

template <int HD, int NQ, bool Q8>
struct PagedShared {
    static constexpr int W = kPagedWaves;
    static constexpr int kHeads = Q8 ? kPagedHeads : 4 * NQ;
    union {
        struct {
            // q as the products take it: fp32 [quad][f] float4 of dims 16 f + 4 g
            // of head 4 quad + i at 4 g + i; 8 bits [s][j] digits j of dims 64 s +
            // 16 g of head m at 16 g + m
            u32x4 q[Q8 ? HD / 16 * kWave : NQ * (HD / 16) * 16];
            alignas(16) float k_new[HD], v_new[HD];  // the new rows (8 bits: of bytes)
            float new_scale[2], q_unit[kPagedHeads];
            float p[Q8 ? 1 : W][Q8 ? 1 : NQ][32][4];  // fp32: a tile's probabilities, by position and head of a quad
        };
        float o[W][kHeads][HD + 4];  // the waves' outputs
        struct {
            float w[kPagedHeads][kPagedSplits + 1];  // the merge: weights of a head's records
            float4 part[W * kWave];                  // and partial sums of them
        } merge;
    };
    struct alignas(16) {
        float m, l;
        int unit;  // 8 bits: the exponent of O's unit
    } sums[W][kPagedHeads];  // the waves' references and sums
    int last;
};

// Over the 16 lanes of a row, and over a wave; the result in every lane.
__device__ __forceinline__ float row_max(float x)
{
    x = fmaxf(x, dpp<0x121>(x));
    x = fmaxf(x, dpp<0x122>(x));
    x = fmaxf(x, dpp<0x124>(x));
    return fmaxf(x, dpp<0x128>(x));
}
__device__ __forceinline__ float row_sum(float x)
{
    x += dpp<0x121>(x);
    x += dpp<0x122>(x);
    x += dpp<0x124>(x);
    return x + dpp<0x128>(x);
}
__device__ __forceinline__ float lanes_max(float x) { return rows4<true>(row_max(x)); }
__device__ __forceinline__ unsigned wave_max_u32(unsigned x) { return rows4_bits(dpp_max16(x)); }
__device__ __forceinline__ float lanes_sum(float x) { return rows4<false>(row_sum(x)); }

// The sum of a group's records by T threads: record s of head h counts
// 2^(lse_s - max lse) / their sum.
template <int HD, int T, typename Merge>
__device__ __forceinline__ void paged_merge(const PagedArgs &a, Merge &sh, size_t first, int n_split, const PagedPlace &p, int tid)
{
    constexpr int LR = HD / 4;
    const int lane = tid & (kWave - 1), items = a.group * LR;
    const size_t rec0 = first * a.group;
    int parts = 1;
    while (2 * parts * items <= T) parts *= 2;
    const int part = parts > 1 ? tid / items : 0;
    const auto wr = make_rsrc(a.ws_o + rec0 * HD, (uint32_t)(n_split * items) * 16u);
    float4 x[8];
    auto load = [&](int i, int s) {  // (past the last record: 0)
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = buf_load4<kSc1>(wr, (uint32_t)((s + k * parts) * items + i) * 16u);
    };
    load(tid - part * items, part);  // on their way while the weights are formed
    const auto lr = make_rsrc(a.ws_lse + rec0, (uint32_t)(n_split * a.group) * 4u);
    for (int head = tid / kWave; head < a.group; head += T / kWave) {
        float y = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(lr, (lane * a.group + head) * 4, 0, kSc1));
        if (lane >= n_split) y = -__builtin_inff();
        y = fast_exp2(y - lanes_max(y));
        sh.w[head][lane] = y * (1.0f / lanes_sum(y));
    }
    __syncthreads();
    float4 *out = reinterpret_cast<float4 *>(a.out) + ((size_t)p.seq * a.n_heads + p.kvh * a.group) * LR;
    for (int i0 = 0; i0 < items; i0 += T) {
        const int i = i0 + tid - part * items, head = i / LR;
        const bool mine = i < items && part < parts;
        float4 acc = make_float4(0, 0, 0, 0);
        for (int s = part; s < n_split; s += 8 * parts) {
            if (i0 > 0 || s != part) load(i, s);
            if (mine)
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (s + k * parts < n_split) fma4(acc, sh.w[head][s + k * parts], x[k]);
        }
        if (parts > 1) {
            sh.part[tid] = acc;
            __syncthreads();
            if (part == 0 && mine)
                for (int t = 1; t < parts; t++) fma4(acc, 1.0f, sh.part[t * items + i]);
        }
        if (part == 0 && mine) out[i] = acc;
    }
}

// ---- fixed-point digits ---------------------------------------------------------

// x of magnitude under 2^30 (already scaled) as four signed digits of 8 bits,
// least first, in the bytes of a word.
__device__ __forceinline__ unsigned digits_of(float x)
{
    return ((unsigned)(int)rintf(x) + 0x80808080u) ^ 0x80808080u;
}
// Digit j of four words, in order: d[j] holds the bytes j of w0..w3.
__device__ __forceinline__ void digits4(unsigned w0, unsigned w1, unsigned w2, unsigned w3, unsigned d[4])
{
    const unsigned a = __builtin_amdgcn_perm(w1, w0, 0x05010400u), b = __builtin_amdgcn_perm(w3, w2, 0x05010400u);
    const unsigned c = __builtin_amdgcn_perm(w1, w0, 0x07030602u), e = __builtin_amdgcn_perm(w3, w2, 0x07030602u);
    d[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    d[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    d[2] = __builtin_amdgcn_perm(e, c, 0x05040100u);
    d[3] = __builtin_amdgcn_perm(e, c, 0x07060302u);
}
// The exponent of a largest magnitude `bits`, at least `least`: what is scaled
// by 2^(29 - e) is below 2^30.
constexpr int kLeastQ = -90, kLeastWeight = -97;  // (2^(29 - e) is a float)
__device__ __forceinline__ int fixed_exp(unsigned bits, int least) { return max((int)(bits >> 23) - 127, least); }
// The four digits' sums together.
__device__ __forceinline__ float digits_sum(int d0, int d1, int d2, int d3)
{
    return __builtin_fmaf((float)((int)((unsigned)d3 << 8) + d2), 65536.0f, (float)((int)((unsigned)d1 << 8) + d0));
}
// The integer at or below a difference of references.
__device__ __forceinline__ int whole_part(float x) { return (int)floorf(fmaxf(x, -1000.0f)); }
__device__ __forceinline__ i32x4 mfma8(u32x4 a, u32x4 b, i32x4 c)
{
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// The smaller / larger; NaN if either is.
__device__ __forceinline__ float4 min4(float4 a, float4 b)
{
    return make_float4(__builtin_elementwise_minimum(a.x, b.x), __builtin_elementwise_minimum(a.y, b.y),
                       __builtin_elementwise_minimum(a.z, b.z), __builtin_elementwise_minimum(a.w, b.w));
}
__device__ __forceinline__ float4 max4(float4 a, float4 b)
{
    return make_float4(__builtin_elementwise_maximum(a.x, b.x), __builtin_elementwise_maximum(a.y, b.y),
                       __builtin_elementwise_maximum(a.z, b.z), __builtin_elementwise_maximum(a.w, b.w));
}
__device__ __forceinline__ float4 shfl_xor4(float4 x, int by)
{
    return make_float4(__shfl_xor(x.x, by), __shfl_xor(x.y, by), __shfl_xor(x.z, by), __shfl_xor(x.w, by));
}
// Four int8 values of a word times a scale.
__device__ __forceinline__ float4 bytes4(int q, float s)
{
    return make_float4((float)(int8_t)q * s, (float)(int8_t)(q >> 8) * s, (float)(int8_t)(q >> 16) * s, (float)(q >> 24) * s);
}

// The least and the largest of each element over a page's keys of one KV head,
// by one wave, LR lanes a row: rows [0, n) from memory, and x (the lane's
// float4 of the row behind them) where more is set.
template <int HD, bool Q8>
__device__ __forceinline__ void page_bounds(const void *k, const float *ks, float *to, int n, float4 x, bool more, int lane)
{
    constexpr int LR = HD / 4, PER = kWave / LR;
    const int c = lane & (LR - 1);
    const float inf = __builtin_inff();
    float4 lo = make_float4(inf, inf, inf, inf), hi = make_float4(-inf, -inf, -inf, -inf);
    if (more) lo = hi = x;
#pragma unroll 4
    for (int r = lane / LR; r < n; r += PER) {
        float4 y;
        if constexpr (Q8)
            y = bytes4(reinterpret_cast<const int *>(k)[r * LR + c], ks[r]);
        else
            y = reinterpret_cast<const float4 *>(k)[r * LR + c];
        lo = min4(lo, y);
        hi = max4(hi, y);
    }
    for (int by = LR; by < kWave; by *= 2) {
        lo = min4(lo, shfl_xor4(lo, by));
        hi = max4(hi, shfl_xor4(hi, by));
    }
    if (lane < LR) {
        reinterpret_cast<float4 *>(to)[c] = lo;
        reinterpret_cast<float4 *>(to)[LR + c] = hi;
    }
}

// Positions of a wave's tile, 16 KiB of fp32 rows and 16 (8 at head_dim 64) of
// 8-bit ones.
__host__ __device__ constexpr int paged_tile(int hd, bool q8) { return q8 ? 64 : 2048 / hd; }

// A row's value of lane j of each row of 16 lanes (DPP row_newbcast).
template <int J>
__device__ __forceinline__ float row_lane(float x)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x150 + J, 0xF, 0xF, true));
}
template <int I, int N, class F>
__device__ __forceinline__ void unroll(F f)
{
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        unroll<I + 1, N>(f);
    }
}

// A run of a group's tiles: [t0, t1) of group gi, run `run` of n, whose
// records start at rec0.  FLAT: all known; else t0 is, and t1 and n follow from
// the position.
struct PagedRun {
    int gi, t0, t1, run, n;
    size_t rec0;
};
// Loads go out before the position is known where that is possible: a run's
// pages do not depend on it.
template <int HD, int NQ, bool Q8, bool FLAT>
__device__ __forceinline__ void paged_run(const PagedArgs &a, PagedShared<HD, NQ, Q8> &sh, const PagedRun &r, int pos)
{
    constexpr int TK = paged_tile(HD, Q8), NB = TK / 16, LR = HD / 4, VB = HD / 16, W = kPagedWaves, kThreads = W * kWave;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int m = lane & 15, g = lane >> 4;
    PagedPlace p = paged_place(a, r.gi);
    const int blocks_log2 = a.rows_log2 - 4;  // blocks of 16 rows of a page
    auto row0_of = [&](int page, int block) {  // a block's first row among the KV heads' rows of the layer
        return (((size_t)page * a.n_kv_heads + p.kvh) << a.rows_log2) + ((block & ((1 << blocks_log2) - 1)) << 4);
    };
    auto there = [&](int page) { return (unsigned)page < (unsigned)a.n_pages; };
    const int t0 = r.t0;
    int t = t0 + wave;

    // ---- a tile's loads ----
    // (always made, on or not, so that the waits for them count exactly: an
    // empty range reads nothing)
    // (blocks behind a sequence's last: page 0 or another's rows, which are masked)
    constexpr int KF = Q8 ? HD / 64 : HD / 16, VR = kWave / LR, VS = 16 / VR;  // (rows of a V load, and loads of a block)
    float4 kraw[Q8 ? 1 : NB][KF], vraw[Q8 ? 1 : NB][Q8 ? 1 : VS];  // fp32
    u32x4 k8[Q8 ? NB : 1][KF], v8[Q8 ? VB : 1];               // 8 bits
    float ksc = 0.0f, vsc = 0.0f;                             // and the scales of position 16 g + m
    // Its pages, a tile ahead.  fp32: of each block, the same in all lanes.  8
    // bits: of blocks m / 4 and g: K's row m of product block b is row 4 b + m
    // % 4 of block m / 4, so that the scores of a lane, 4 for each b, are the
    // 16 rows of block g in order, which are the 16 bytes of V that it loads.
    int pages[Q8 ? 2 : NB];
    auto look = [&](int at) {
        if constexpr (Q8) {
            int here = lane;
            asm volatile("" : "+v"(here));
            pages[0] = p.list[min(4 * at + ((here & 15) >> 2), a.blocks - 1) >> blocks_log2];
            pages[1] = p.list[min(4 * at + (here >> 4), a.blocks - 1) >> blocks_log2];
        } else {
#pragma unroll
            for (int b = 0; b < NB; b++) pages[b] = uniform_load(p.list + (min(at * NB + b, a.blocks - 1) >> blocks_log2));
        }
    };
    const int8_t *v8_at = nullptr;
    const float *vs_at = nullptr;
    int used[Q8 ? 1 : NB];  // fp32: the pages of the tile that is loaded
    auto load_k = [&](int at, bool on) {
        if constexpr (Q8) {
            int here = on ? lane : 0;  // (not on: all lanes the same line)
            asm volatile("" : "+v"(here));  // (addresses formed here: kept, their parts would take the registers of a load)
            const int m = here & 15, g = here >> 4;
            const size_t rk = row0_of(on && there(pages[0]) ? pages[0] : 0, 4 * at + (m >> 2)) + (m & 3);
            const size_t rv = row0_of(on && there(pages[1]) ? pages[1] : 0, 4 * at + g);
            const int8_t *from = static_cast<const int8_t *>(a.k) + rk * HD + 16 * g;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int s = 0; s < KF; s++)
                    k8[b][s] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(from + 4 * b * HD + 64 * s));
            ksc = a.ks[rv + m];
            v8_at = static_cast<const int8_t *>(a.v) + rv * HD + 16 * m;
            vs_at = a.vs + rv + m;
        } else {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                used[b] = pages[b];
                const bool ok = on && there(pages[b]);
                const auto rows = make_rsrc(static_cast<const float *>(a.k) + row0_of(ok ? pages[b] : 0, at * NB + b) * HD, ok ? 64u * HD : 0u);
#pragma unroll
                for (int f = 0; f < KF; f++) kraw[b][f] = buf_load4<kNt>(rows, (uint32_t)(m * HD + 16 * f + 4 * g) * 4u);
            }
        }
    };
    auto load_v = [&](int at, bool on) {
        if constexpr (Q8) {
#pragma unroll
            for (int v = 0; v < VB; v++) v8[v] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(v8_at + 256 * v));
            vsc = *vs_at;
        } else {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const bool ok = on && there(used[b]);
                const auto rows = make_rsrc(static_cast<const float *>(a.v) + row0_of(ok ? used[b] : 0, at * NB + b) * HD, ok ? 64u * HD : 0u);
#pragma unroll
                for (int v = 0; v < VS; v++) vraw[b][v] = buf_load4<kNt>(rows, (uint32_t)(v * VR * HD + 4 * lane) * 4u);
            }
        }
    };
    // ---- rows of q, and the new token's ----
    // LR lanes a row, by the first waves alone: a CU's loads come back in the
    // order in which its waves made them, and everyone waits for q.  These
    // loads, the position's and the first pages' go out together.  (A head
    // that the group leaves out is zero.)
    const int c = lane & (LR - 1);
    constexpr int kPer = kWave / LR, kHeads = Q8 ? kPagedHeads : 4 * NQ;       // rows of a wave at a time, and of q
    constexpr int kRows = (kHeads + W * kPer - 1) / (W * kPer);
    constexpr int kRowWaves = (kHeads + kRows * kPer - 1) / (kRows * kPer);    // waves that have some
    static_assert(kHeads % (kRows * kPer) == 0 || kRowWaves == 1, "rows of q");
    const int head0 = wave * kRows * kPer + lane / LR;
    const size_t new_at = ((size_t)p.seq * a.n_kv_heads + p.kvh) * LR;
    const bool has_rows = wave < kRowWaves && wave * kRows * kPer < a.group;
    if (has_rows) __builtin_amdgcn_s_setprio(3);
    float4 row[kRows];
    const auto q_rows = make_rsrc(a.q + ((size_t)p.seq * a.n_heads + p.kvh * a.group) * HD, has_rows ? (uint32_t)(a.group * HD) * 4u : 0u);
#pragma unroll
    for (int u = 0; u < kRows; u++) row[u] = buf_load4(q_rows, (uint32_t)((head0 + u * kPer) * LR + c) * 16u);
    const uint32_t new_bytes = wave == 0 ? HD * 4u : 0u;
    const float4 k_row = buf_load4(make_rsrc(a.k_new + new_at * 4, new_bytes), c * 16u);
    const float4 v_row = buf_load4(make_rsrc(a.v_new + new_at * 4, new_bytes), c * 16u);
    look(t);
    p.pos = FLAT ? pos : uniform_load(a.pos + p.seq);
    const int whole = FLAT ? 0x7fffffff : uniform_load(a.whole + p.seq);
    if constexpr (!Q8) asm volatile("" ::"s"(p.pos), "s"(whole), "s"(pages[0]), "s"(pages[NB - 1]));  // (one wait for them all)
    __builtin_amdgcn_sched_barrier(0);
    paged_rows(a, p, whole);
    if (!FLAT && p.skip) {
        if (r.run == 0) paged_skip<HD>(a, p, tid);
        return;
    }
    const int tiles = (p.rows + TK - 1) / TK;
    if (!FLAT && t0 >= tiles) return;
    const int t1 = FLAT ? r.t1 : min(t0 + a.chunk, tiles), n_runs = FLAT ? r.n : paged_runs(a, tiles), n_blocks = (p.rows + 15) >> 4;
    const bool newest_run = t1 == tiles;
    const float4 turn = buf_load4(make_rsrc(a.rope + (size_t)p.pos * LR, has_rows ? HD * 4u : 0u), c * 16u);
    __builtin_amdgcn_sched_barrier(0);
    load_k(t, t < t1);
    load_v(t, t < t1);
    look(t + W);
    __builtin_amdgcn_sched_barrier(0);
    auto put_row = [&](int job, float4 x) {
        if constexpr (Q8) {
            unsigned top = dpp_max16(max4_bits(0u, x));
            if constexpr (HD == 128) top = max(top, (unsigned)__shfl_xor((int)top, 16));
            const bool good = finite_bits(top);
            const int e = fixed_exp(good ? top : 0u, kLeastQ);
            const float up = good ? exp2_int(29 - e) : 0.0f;
            unsigned d[4];
            digits4(digits_of(x.x * up), digits_of(x.y * up), digits_of(x.z * up), digits_of(x.w * up), d);
            // dims 4 c: s = c / 16, g = c / 4 % 4, word c % 4
#pragma unroll
            for (int j = 0; j < 4; j++) reinterpret_cast<unsigned *>(&sh.q[(4 * (c >> 4) + j) * kWave + 16 * ((c >> 2) & 3) + job])[c & 3] = d[j];
            if (c == 0) sh.q_unit[job] = good ? exp2_int(e - 29) * a.scale_log2 : __uint_as_float(0x7fc00000u);
        } else {
            // dims 4 c: f = c / 4, g = c % 4
            sh.q[((job >> 2) * (HD / 16) + (c >> 2)) * 16 + 4 * (c & 3) + (job & 3)] = u32x4{__float_as_uint(x.x), __float_as_uint(x.y), __float_as_uint(x.z), __float_as_uint(x.w)};
        }
    };
    if (has_rows) {
#pragma unroll
        for (int u = 0; u < kRows; u++) put_row(head0 + u * kPer, rope4(row[u], turn));
    } else if (wave < kRowWaves) {
#pragma unroll
        for (int u = 0; u < kRows; u++) put_row(head0 + u * kPer, make_float4(0, 0, 0, 0));
    }
    if (newest_run && wave == 0) {
        const float4 x[2] = {rope4(k_row, turn), v_row};
#pragma unroll
        for (int value = 0; value < 2; value++) {
            float *to = value ? sh.v_new : sh.k_new;
            if constexpr (Q8) {
                float sc;
                const int w = quantize_row<HD>(x[value], &sc);
                reinterpret_cast<int *>(to)[c] = w;
                if (c == 0) sh.new_scale[value] = sc;
            } else {
                reinterpret_cast<float4 *>(to)[c] = x[value];
            }
        }
    }
    if (has_rows) __builtin_amdgcn_s_setprio(0);
    __syncthreads();
    const float qf = Q8 ? sh.q_unit[m] : a.scale_log2;

    // ---- the new rows into the cache, by the wave that has the last tile ----
    const bool has_new = newest_run && (tiles - 1 - t0) % W == wave;
    const int new_row = (p.rows - 1) & (TK - 1);                       // its row of the last tile
    const int b_new = new_row >> 4, r_new = new_row & 15;              // its block of that, and row of the block
    bool shared = false;  // the new row's page is not the sequence's own
    if (has_new) {
        const int own = uniform_load(p.list + p.n_list - 1);
        shared = !there(own) || uniform_load(a.refs + (there(own) ? own : 0)) != 1;
        if (!shared && lane < LR) {
            const size_t to = row0_of(own, n_blocks - 1) + r_new;
            if constexpr (Q8) {
                const int w = reinterpret_cast<const int *>(sh.v_new)[lane];
                reinterpret_cast<int *>(a.k)[to * LR + lane] = reinterpret_cast<const int *>(sh.k_new)[lane];
                int8_t *bytes = static_cast<int8_t *>(a.v) + (to - r_new) * HD + 64 * lane + r_new;
#pragma unroll
                for (int i = 0; i < 4; i++) bytes[16 * i] = (int8_t)(w >> (8 * i));
                if (lane == 0) {
                    a.ks[to] = sh.new_scale[0];
                    a.vs[to] = sh.new_scale[1];
                }
            } else {
                reinterpret_cast<float4 *>(a.k)[to * LR + lane] = reinterpret_cast<const float4 *>(sh.k_new)[lane];
                reinterpret_cast<float4 *>(a.v)[to * LR + lane] = reinterpret_cast<const float4 *>(sh.v_new)[lane];
            }
        }
        if (!shared && a.bounds && (p.pos & ((1 << a.rows_log2) - 1)) == (1 << a.rows_log2) - 1) {
            // the page is complete: the bounds of its keys
            const size_t head = (size_t)own * a.n_kv_heads + p.kvh;
            const int d = lane & (LR - 1);
            const float4 x = Q8 ? bytes4(reinterpret_cast<const int *>(sh.k_new)[d], sh.new_scale[0])
                                : reinterpret_cast<const float4 *>(sh.k_new)[d];
            page_bounds<HD, Q8>(static_cast<const char *>(a.k) + (head << a.rows_log2) * HD * (Q8 ? 1 : 4),
                                Q8 ? a.ks + (head << a.rows_log2) : nullptr, a.bounds + head * 2 * HD, (1 << a.rows_log2) - 1, x, true,
                                lane);
        }
    }

    // fp32: o[4 quad + e] has dims 4 (lane % LR) + e of the quad's heads, over
    // the rows lane / LR of each V load; a lane's sums are of head 4 quad + g.
    // 8 bits: o[v] has dims 16 v + 4 g + i of head m, and the sums are of head m.
    constexpr int kAcc = Q8 ? VB : 4 * NQ, kSums = Q8 ? 1 : NQ;
    f32x4 o[kAcc];
#pragma unroll
    for (int v = 0; v < kAcc; v++) o[v] = f32x4{0, 0, 0, 0};
    float mrun[kSums], lrun[kSums];
    int unit = kLeastWeight;
#pragma unroll
    for (int k = 0; k < kSums; k++) {
        mrun[k] = kNothing;
        lrun[k] = 0.0f;
    }
    for (; t < t1; t += W) {
        const bool last = t == tiles - 1, next = t + W < t1;
        int zero = 0;
        asm volatile("" : "+v"(zero));  // (q is read from LDS for each tile: kept, it would take a quarter of the registers)
        if constexpr (!Q8) {
            if (last) {
#pragma unroll
                for (int b = 0; b < NB; b++)
                    if (b == b_new && m == r_new)
#pragma unroll
                        for (int f = 0; f < KF; f++) kraw[b][f] = *reinterpret_cast<const float4 *>(&sh.k_new[16 * f + 4 * g]);
            }
            // ---- scores ----
            const u32x4 *qs = &sh.q[4 * g + (m & 3) + zero];
            float x[NQ][NB];  // of head 4 quad + g at position 16 b + m
            f32x4 s[NQ][NB][2];
#pragma unroll
            for (int k = 0; k < NQ; k++)
#pragma unroll
                for (int b = 0; b < NB; b++) s[k][b][0] = s[k][b][1] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int f = 0; f < KF; f++)
#pragma unroll
                for (int k = 0; k < NQ; k++) {
                    const f32x4 q = __builtin_bit_cast(f32x4, qs[(k * KF + f) * 16]);
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        s[k][b][0] = __builtin_amdgcn_mfma_f32_4x4x1f32(q.x, kraw[b][f].x, s[k][b][0], 0, 0, 0);
                        s[k][b][1] = __builtin_amdgcn_mfma_f32_4x4x1f32(q.y, kraw[b][f].y, s[k][b][1], 0, 0, 0);
                        s[k][b][0] = __builtin_amdgcn_mfma_f32_4x4x1f32(q.z, kraw[b][f].z, s[k][b][0], 0, 0, 0);
                        s[k][b][1] = __builtin_amdgcn_mfma_f32_4x4x1f32(q.w, kraw[b][f].w, s[k][b][1], 0, 0, 0);
                    }
                }
            load_k(t + W, next);
            // ---- softmax ----
            float up = -__builtin_inff();
#pragma unroll
            for (int k = 0; k < NQ; k++)
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const f32x4 y = s[k][b][0] + s[k][b][1];
                    x[k][b] = halves_sum2(rows_sum2(y[0], y[1]), rows_sum2(y[2], y[3])) * a.scale_log2;
                    if (last && 16 * b + m > new_row) x[k][b] = -__builtin_inff();
                    up = fmaxf(up, x[k][b] - mrun[k]);
                }
            if (__builtin_amdgcn_ballot_w64(up > kPagedMargin) != 0) {
#pragma unroll
                for (int k = 0; k < NQ; k++) {
                    float mt = x[k][0];
#pragma unroll
                    for (int b = 1; b < NB; b++) mt = fmaxf(mt, x[k][b]);
                    mt = row_max(mt);
                    const float now = mt > mrun[k] + kPagedMargin ? mt : mrun[k], f = fast_exp2(mrun[k] - now);
                    mrun[k] = now;
                    lrun[k] *= f;
                    const f32x4 by = {lane_value(f, 0), lane_value(f, 16), lane_value(f, 32), lane_value(f, 48)};
#pragma unroll
                    for (int e = 0; e < 4; e++) o[4 * k + e] *= by;
                }
            }
#pragma unroll
            for (int k = 0; k < NQ; k++)
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    x[k][b] = fast_exp2(x[k][b] - (mrun[k] + kPagedBias<Q8>));
                    lrun[k] += x[k][b];
                    sh.p[wave][k][16 * b + m][g] = x[k][b];
                }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (last) {
                // the new value, and zeros behind it
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int v = 0; v < VS; v++) {
                        const int row = 16 * b + VR * v + lane / LR;
                        if (row >= new_row)
                            vraw[b][v] = row == new_row ? *reinterpret_cast<const float4 *>(&sh.v_new[4 * (lane & (LR - 1))])
                                                      : make_float4(0, 0, 0, 0);
                    }
            }
            // ---- weighted values ----
#pragma unroll
            for (int k = 0; k < NQ; k++)
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int v = 0; v < VS; v++) {
                        const float w = sh.p[wave][k][16 * b + VR * v + lane / LR][lane & 3];
                        o[4 * k] = __builtin_amdgcn_mfma_f32_4x4x1f32(w, vraw[b][v].x, o[4 * k], 0, 0, 0);
                        o[4 * k + 1] = __builtin_amdgcn_mfma_f32_4x4x1f32(w, vraw[b][v].y, o[4 * k + 1], 0, 0, 0);
                        o[4 * k + 2] = __builtin_amdgcn_mfma_f32_4x4x1f32(w, vraw[b][v].z, o[4 * k + 2], 0, 0, 0);
                        o[4 * k + 3] = __builtin_amdgcn_mfma_f32_4x4x1f32(w, vraw[b][v].w, o[4 * k + 3], 0, 0, 0);
                    }
        } else {
            const u32x4 *qs = &sh.q[lane + zero];
            const bool first = t == t0 + wave;  // (o is zero)
            float x[NB][4], mt = -__builtin_inff();
            if (last) {
#pragma unroll
                for (int b = 0; b < NB; b++)
                    if (4 * b + (m & 3) == r_new && (m >> 2) == b_new)
#pragma unroll
                        for (int s = 0; s < KF; s++)
                            k8[b][s] = *reinterpret_cast<const u32x4 *>(reinterpret_cast<const int8_t *>(sh.k_new) + 64 * s + 16 * g);
                if (g == b_new && m == r_new) {
                    ksc = sh.new_scale[0];
                    vsc = sh.new_scale[1];
                }
            }
            // ---- scores ----
            // (NaN in either of a row's scales marks it)
            const float sc = ksc + 0.0f * vsc;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                i32x4 d[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    d[j] = i32x4{0, 0, 0, 0};
#pragma unroll
                    for (int s = 0; s < KF; s++) d[j] = mfma8(k8[b][s], qs[(4 * s + j) * kWave], d[j]);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) x[b][i] = digits_sum(d[0][i], d[1][i], d[2][i], d[3][i]) * qf;
                // (put together here: all sums of a tile at once would not fit the registers)
                asm volatile("" : "+v"(x[b][0]), "+v"(x[b][1]), "+v"(x[b][2]), "+v"(x[b][3]));
            }
            unroll<0, 16>([&](auto j) { x[j / 4][j % 4] *= row_lane<j>(sc); });
            if (last) {
                // the new value's byte of each dim's 16
                const int sh8 = 8 * (r_new & 3);
                const uint8_t *y = reinterpret_cast<const uint8_t *>(sh.v_new);
#pragma unroll
                for (int v = 0; v < VB; v++) {
                    const unsigned w = (unsigned)y[16 * v + m] << sh8;
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (g == b_new && i == (r_new >> 2)) v8[v][i] = (v8[v][i] & ~(255u << sh8)) | w;
                }
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (16 * g + 4 * b + i > new_row) x[b][i] = -__builtin_inff();
            }
            load_k(t + W, next);
            __builtin_amdgcn_sched_barrier(0);
            // ---- softmax ----
#pragma unroll
            for (int b = 0; b < NB; b++) mt = fmaxf(mt, fmaxf(fmaxf(x[b][0], x[b][1]), fmaxf(x[b][2], x[b][3])));
            if (__builtin_amdgcn_ballot_w64(mt > mrun[0] + kPagedMargin) != 0) {
                mt = rows4<true>(mt);
                const float now = mt > mrun[0] + kPagedMargin ? mt : mrun[0], d = mrun[0] - now;
                const int down = max(unit + whole_part(d), kLeastWeight);  // (O's unit goes with its weights)
                const float f = fast_exp2(d - (float)(down - unit));
                mrun[0] = now;
                lrun[0] *= fast_exp2(d);
                unit = down;
                if (!first)
#pragma unroll
                    for (int v = 0; v < VB; v++) o[v] *= f;
            }
            const float off = mrun[0] + kPagedBias<Q8>, vs = fmaxf(vsc, 0.0f);
            float wt = 0.0f;
            unroll<0, 16>([&](auto j) {
                const float y = fast_exp2(x[j / 4][j % 4] - off);
                lrun[0] += y;
                x[j / 4][j % 4] = y * row_lane<j>(vs);
                wt = fmaxf(wt, x[j / 4][j % 4]);
            });
            // ---- weighted values ----
            const int e = fixed_exp(__float_as_uint(rows4<true>(wt)), kLeastWeight);
            if (__builtin_amdgcn_ballot_w64(e > unit) != 0) {
                const int now = max(unit, min(e + 2, 127));
                const float f = exp2_int(max(unit - now, -126));
                unit = now;
                if (!first)
#pragma unroll
                    for (int v = 0; v < VB; v++) o[v] *= f;
            }
            const float up = exp2_int(29 - e), down = exp2_int(max(e - unit - 29, -126));
            u32x4 pd[4];
#pragma unroll
            for (int b = 0; b < NB; b++) {
                unsigned d[4];
                digits4(digits_of(x[b][0] * up), digits_of(x[b][1] * up), digits_of(x[b][2] * up), digits_of(x[b][3] * up), d);
#pragma unroll
                for (int j = 0; j < 4; j++) pd[j][b] = d[j];
            }
#pragma unroll
            for (int v = 0; v < VB; v++) {
                i32x4 d[4];
#pragma unroll
                for (int j = 0; j < 4; j++) d[j] = mfma8(v8[v], pd[j], i32x4{0, 0, 0, 0});
#pragma unroll
                for (int i = 0; i < 4; i++) o[v][i] = __builtin_fmaf(digits_sum(d[0][i], d[1][i], d[2][i], d[3][i]), down, o[v][i]);
                v8[v] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(v8_at + 256 * v));  // (the next tile's)
                asm volatile("" : "+v"(o[v]));
                __builtin_amdgcn_sched_barrier(0);
            }
            vsc = *vs_at;
        }
        if constexpr (!Q8) load_v(t + W, next);
        look(t + 2 * W);
    }

    // ---- the waves' results together ----
    __syncthreads();  // (q is read; its memory takes the outputs)
    if constexpr (Q8) {
        const float l = rows4<false>(lrun[0]);
        if (g == 0) {
            sh.sums[wave][m].m = mrun[0];
            sh.sums[wave][m].unit = unit;
            sh.sums[wave][m].l = shared ? __uint_as_float(0x7fc00000u) : l;
        }
        if (m < a.group)
#pragma unroll
            for (int v = 0; v < VB; v++)
                *reinterpret_cast<float4 *>(&sh.o[wave][m][16 * v + 4 * g]) = make_float4(o[v][0], o[v][1], o[v][2], o[v][3]);
    } else {
#pragma unroll
        for (int k = 0; k < NQ; k++) {
            const float l = row_sum(lrun[k]);
            if (m == 0) {
                sh.sums[wave][4 * k + g].m = mrun[k];
                sh.sums[wave][4 * k + g].l = shared ? __uint_as_float(0x7fc00000u) : l;
            }
        }
        f32x4 acc[NQ][4];
#pragma unroll
        for (int k = 0; k < NQ; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[k][e] = o[4 * k + e];
        slot_sums<HD, 4 * NQ>(acc, lane, [&](int, int head, float4 y) {
            *reinterpret_cast<float4 *>(&sh.o[wave][head][4 * (lane & (LR - 1))]) = y;
        });
    }
    __syncthreads();
    const size_t rec = (r.rec0 + r.run) * a.group;
    for (int i = tid; i < a.group * LR; i += kThreads) {
        const int head = i / LR, d = (i - head * LR) * 4;
        std::remove_reference_t<decltype(sh.sums[0][0])> part[W];
#pragma unroll
        for (int w = 0; w < W; w++) part[w] = sh.sums[w][head];
        float top = part[0].m;
#pragma unroll
        for (int w = 1; w < W; w++) top = fmaxf(top, part[w].m);
        float f[W], total = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) {
            f[w] = fast_exp2(part[w].m - top);
            total += f[w] * part[w].l;
        }
        float o_unit = 1.0f;
        if constexpr (Q8) {
            // in the largest of the waves' units, as they count
            int unit = kLeastWeight;
#pragma unroll
            for (int w = 0; w < W; w++) unit = max(unit, part[w].unit + whole_part(part[w].m - top));
#pragma unroll
            for (int w = 0; w < W; w++) f[w] = fast_exp2(part[w].m - top + (float)(part[w].unit - unit));
            o_unit = exp2_int(unit);
        }
        float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < W; w++) fma4(acc, f[w], *reinterpret_cast<const float4 *>(&sh.o[w][head][d]));
        // (no weight at all, every score -inf: as a record nothing, as a result NaN)
        if (n_runs == 1) {
            scale4(acc, 1.0f / total);
            if constexpr (Q8) scale4(acc, o_unit);
            *reinterpret_cast<float4 *>(a.out + ((size_t)p.seq * a.n_heads + p.kvh * a.group + head) * HD + d) = acc;
        } else {
            scale4(acc, total == 0.0f ? 0.0f : 1.0f / total);
            if constexpr (Q8) scale4(acc, o_unit);
            *reinterpret_cast<float4 *>(a.ws_o + (rec + head) * HD + d) = acc;
            if (d == 0) a.ws_lse[rec + head] = total == 0.0f ? -__builtin_inff() : top + log2f(total);
        }
    }
    if (n_runs == 1 || a.spread) return;

    // ---- the last run to arrive adds up the records ----
    // (all in one XCD's L2: the stores have drained to it, the counter is an
    // L2 atomic, and the loads miss in L1)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
        const int before = __hip_atomic_fetch_add(a.counters + (size_t)r.gi * kCtrStride, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sh.last = before == n_runs - 1;
        if (before == n_runs - 1) __hip_atomic_store(a.counters + (size_t)r.gi * kCtrStride, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (sh.last) paged_merge<HD, kThreads>(a, sh.merge, r.rec0, n_runs, p, tid);
}

// (waves a SIMD: fp32 rows on their way in as many as the registers allow)
__host__ __device__ constexpr int paged_occupancy(int nq, bool q8) { return q8 ? 3 : nq == 1 ? 4 : nq == 2 ? 3 : 2; }

// Runs of equal length, the same number for every group, which short ones do
// not use up.
template <int HD, int NQ, bool Q8>
__global__ __launch_bounds__(kPagedWaves *kWave, paged_occupancy(NQ, Q8)) void paged_attention_kernel(PagedArgs a)
{
    __shared__ PagedShared<HD, NQ, Q8> sh;
    // the group and its run: a group's runs on one XCD, or (spread) on all
    const int n_groups = a.n_seq * a.n_kv_heads;
    int gi, run;
    if (a.spread) {
        run = (int)fast_div(blockIdx.x, a.by_groups);
        gi = blockIdx.x - run * n_groups;
    } else {
        const int local = blockIdx.x / kXcds, gl = (int)fast_div((uint32_t)local, a.by_splits);
        run = local - gl * a.splits;
        gi = gl * kXcds + (blockIdx.x & (kXcds - 1));
    }
    if (gi >= n_groups) return;
    paged_run<HD, NQ, Q8, false>(a, sh, PagedRun{gi, run * a.chunk, 0, run, 0, (size_t)gi * a.splits}, 0);
}

// A batch whose groups do not cut evenly: an XCD's groups (i kXcds + its
// number) laid end to end and cut into runs of equal length, one a workgroup,
// which may end one group and begin the next.  A beginning counts as
// kPagedStart tiles.  Records: run w's of group i is w + i of the XCD's (one of
// the two grows from each to the next, so a group's lie together).
constexpr int kPagedStart = 4;
// Tiles and starts of a run, where an XCD's n_wg workgroups share `total`.
__host__ __device__ inline int paged_length(int total, int n_wg)
{
    const int each = (total + n_wg - 1) / n_wg;
    return each > kPagedWaves ? each : kPagedWaves;
}
// Run w's part [t0, t1) of the tiles of an XCD's item (empty: t1 <= t0), the
// run's number among the item's n, and the XCD's record of the item's first.
// The run covers [at, stop), and the item its last len of [0, end).
struct PagedSegment {
    int t0, t1, run, n, record;
};
__host__ __device__ inline PagedSegment paged_segment(int w, int length, int at, int stop, int item, int len, int end)
{
    const int row0 = end - len + kPagedStart, first = row0 / length;
    return {(at > row0 ? at : row0) - row0, (stop < end ? stop : end) - row0, w - first, (end - 1) / length - first + 1, first + item};
}
template <int HD, int NQ, bool Q8>
__global__ __launch_bounds__(kPagedWaves *kWave, NQ == 4 && HD == 64 && !Q8 ? 1 : 2) void paged_flat_kernel(PagedArgs a)
{
    __shared__ PagedShared<HD, NQ, Q8> sh;
    constexpr int TK = paged_tile(HD, Q8);
    const int tid = threadIdx.x, lane = tid & (kWave - 1);
    const int xcd = blockIdx.x & (kXcds - 1), w = blockIdx.x / kXcds, n_wg = gridDim.x / kXcds;
    const int n_groups = a.n_seq * a.n_kv_heads, items = (n_groups - xcd + kXcds - 1) / kXcds;
    // lane i: item i's tiles
    int len = 0, pos = 0;
    if (lane < items) {
        PagedPlace p = paged_place(a, lane * kXcds + xcd);
        p.pos = pos = a.pos[p.seq];
        paged_rows(a, p, a.whole[p.seq]);
        if (!p.skip)
            len = (p.rows + TK - 1) / TK + kPagedStart;
        else if (w == 0 && tid < kWave)
            paged_skip<HD>(a, p, 0, 1);
    }
    const int upto = wave_scan_add(len);
    const int total = __builtin_amdgcn_readlane(upto, kWave - 1);
    const int length = paged_length(total, n_wg), stop = min((w + 1) * length, total);
    bool again = false;
    for (int at = w * length; at < stop;) {
        const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > at));
        const int end = __builtin_amdgcn_readlane(upto, l);
        const PagedSegment s = paged_segment(w, length, at, stop, l, __builtin_amdgcn_readlane(len, l), end);
        if (s.t1 > s.t0) {
            if (again) __syncthreads();  // (the last group's outputs are read)
            again = true;
            paged_run<HD, NQ, Q8, true>(a, sh, PagedRun{l * kXcds + xcd, s.t0, s.t1, s.run, s.n, (size_t)xcd * (n_wg + a.splits) + s.record},
                                        __builtin_amdgcn_readlane(pos, l));
        }
        at = end;
    }
}

// The records of a spread launch's groups added up, a workgroup each.
template <int HD, bool Q8>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedArgs a)
{
    __shared__ struct {
        float w[kPagedHeads][kPagedSplits + 1];
        float4 part[256];
    } sh;
    PagedPlace p = paged_place(a, blockIdx.x);
    p.pos = a.pos[p.seq];
    paged_rows(a, p, a.whole[p.seq]);
    if (p.skip) return;
    const int n_runs = paged_runs(a, (p.rows + paged_tile(HD, Q8) - 1) / paged_tile(HD, Q8));
    if (n_runs > 1) paged_merge<HD, 256>(a, sh, (size_t)blockIdx.x * a.splits, n_runs, p, threadIdx.x);
}

}  // namespace leap
