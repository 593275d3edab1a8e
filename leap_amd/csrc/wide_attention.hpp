// Attention of many rows over a cache: prompts, and trees of more than 16
// (token, q head) rows a KV head.  The rows, products, splits into fp16 halves
// and records are those of many_attention.hpp; here a workgroup of eight
// waves takes a tile of 256 rows, 32 a wave, and the positions of its chunk
// in tiles of 32, split into fp16 halves once, in LDS, for all of them.
//
// Per wave and tile of 32 positions at head_dim 128: 48 32x32x16 MFMAs (three
// products of S^T = K Q^T and of O^T = V^T P^T), 1536 cycles of the matrix
// core, and about 340 vector instructions: 260 of the vector phase (the
// scores' scaling, maximum and 16 exponentials, the split of P, the largest
// magnitudes of a share of the next tile) and that share's split, which fills
// the waits between the products of the matrix phase (in the vector phase it
// took 4 to 10% longer).  The two waves of a SIMD do these in turn: waves 0-3
// are in the matrix phase (the scores of tile i + 1, the weighted values of
// tile i) while waves 4-7 are in the vector phase, a barrier between the
// half-steps.
//
// Half-step h of waves 0-3: scores of tile 0 at h = 0, vector phase i at
// 2 i + 1, matrix phase i at 2 i + 2; waves 4-7 one half-step later.  Waves
// 4-7 bring K: tile i + 2 in matrix phase i (h = 2 i + 3), read from h = 2 (i
// + 2) on, when the buffer's last tile i was read last at h = 2 i + 1: two
// buffers.  Waves 0-3 bring V: tile i + 1 in matrix phase i (h = 2 i + 2),
// read from h = 2 i + 4 to 2 i + 5: three buffers.  The factors are written a
// half-step earlier, K's of tile i + 2 at h = 2 i + 2, V's of tile i + 1 at
// 2 i + 1, and read in vector phases until h = 2 i + 6 and 2 i + 4: four.
//
// Scales: K's and V's exponents by quads of four positions (8-bit caches:
// scales by position).  K's multiply the scores, V's go into the
// probabilities, over O's unit in the row (vrun, next_unit).  A quad with a
// position 2^4 times smaller than another gets an exponent for each, counted in
// its tile's scores and probabilities: so what a row does not see takes no more
// of its accuracy than that.  (Exponents by position throughout took 10 to 20%
// more at 8192 tokens 32/8/128; values over two orders, where most tiles have
// such a quad, take 672 us for 525 at 4096 tokens.)
//
// The softmax reference moves only when a score exceeds it by more than 2^8,
// and O's unit only when a product could pass fp16's range (fits_unit, asked
// of the tile's largest score and factor): such a tile is taken once more, by
// its products.
//
// Measured, heads/KV heads/head_dim: 8192 tokens 32/8/128 in fp32 1671 us with
// their append, 329 TFLOP/s of useful work (987 of fp16 products), the card at
// 1.6 to 2.0 GHz under it; 500 tokens after 6800 64/8/128 374 us (309 TFLOP/s);
// 4096 tokens over an 8-bit cache 310 us (443 TFLOP/s).  A workgroup's start
// (its rows of Q) is about 10 us, its results 2 to 3.
//
// A call of few tokens (fused) has its new rows rotated, quantised and stored
// here, ahead of the first tile.
#pragma once

#include "many_attention.hpp"

namespace leap {

// (the lambdas below are used once or twice each, in a kernel that has no
// registers for calls)
#define LEAP_INLINE __attribute__((always_inline))

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kWideWaves = 8;
constexpr int kWideThreads = kWideWaves * kWave;
constexpr unsigned kUnlike = 4;  // binary orders between positions of a quad from which each has an exponent of its own

template <int HD, bool Q8>
struct WideShared {
    static constexpr int P = Q8 ? 1 : 2;  // halves: high (and low)
    // the low halves of Q of each wave's last kQLow steps, for which there are no registers
    static constexpr int kQLow = HD == 128 ? (Q8 ? 4 : 6) : 0;
    union {
        struct {
            half8v k[2][P][32 * HD / 8];  // [position][dims], 16-byte pieces swizzled by position
            half8v v[3][P][HD * 32 / 8];  // [dim][positions], pieces swizzled by dim
            half8v ql[kWideWaves][kQLow ? kQLow : 1][kWave];
        };
        half8v q[kWideWaves][2][32 * HD / 8];  // first: rows of Q on their way into registers
        float4 o[kWideWaves][32 * HD / 4];     // last: rows of the result on theirs out
    };
    float qf[kWideWaves][32];             // factors of Q's rows
    // factors of K's and V's positions, by lane half: position 8 (j / 4) + 4
    // half + j % 4; fp32: of quads, and of positions only in unlike quads
    float kfac[4][2][16], vfac[4][2][16], kquad[4][2][4], vquad[4][2][4];
    // fp32, by the wave that brought them: positions that are not finite
    // (bits 0-7), quads of unlike positions (bits 8-9); any: of a tile so far
    int odd[4][kWideWaves], any_odd;
    uint64_t sees[kTreeMax], bad;  // tree_lane of each node, and the bad ones
};

__device__ __forceinline__ f32x16 mfma32(half8v a, half8v b, f32x16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// max / sum of a lane's value and the one of the lane 32 away
__device__ __forceinline__ float half_max(float x)
{
    float y = x;
    asm("" : "+v"(y));  // (two registers: the swap of one with itself would be folded)
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

template <int HD, bool Q8>
__global__ __launch_bounds__(kWideThreads, 2) void wide_attention_kernel(ManyArgs a)
{
    constexpr int BM = kWideRows, KS = HD / 16, VB = HD / 32, LR = HD / 4;
    constexpr int C = HD / 8;  // 16-byte pieces of a K row
    __shared__ WideShared<HD, Q8> sh;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int n = lane & 31, g = lane >> 5;
    const bool brings_v = wave < 4;
    const int w = wave & 3;

    // the workgroup's tile, KV head and chunk: neighbouring ids go to other XCDs
    const int n_groups = a.slots * a.n_kv_heads;
    int group_i, split;
    if (a.spread) {
        split = blockIdx.x / n_groups;
        group_i = blockIdx.x - split * n_groups;
    } else {
        split = 0;
        group_i = blockIdx.x;
    }
    if (a.fused && a.begin && blockIdx.x == 0) {
        bool stop = false, any = false;
        for (int base = 0; base < a.n_seq && !stop && !any; base += kWave)
            any = __builtin_amdgcn_ballot_w64(seq_lane(a, base, lane, &stop).n < 0) != 0;
        if (any)
            for (int r = wave; r < a.n_tokens; r += kWideWaves) {
                const TokenPlace t = find_token(a, r, lane);
                if (t.seq >= 0 && t.skip)
                    fill_nan<HD>(a.out, (size_t)r * a.n_heads * LR, a.n_heads * LR, lane, kWave);
            }
    }
    const int slot = (int)fast_div((uint32_t)group_i, a.by_kv_heads);
    const int kvh = group_i - slot * a.n_kv_heads;
    const Place p = find_place<BM>(a, slot, lane);
    if (p.seq < 0) return;
    const int rows = p.n * a.group, r0 = p.tile * BM;
    const int j0 = (int)fast_div((uint32_t)r0, a.by_group);
    const int j1 = min(p.n - 1, (int)fast_div((uint32_t)(r0 + BM - 1), a.by_group));
    const int kv_end = a.parent ? p.p0 + p.n : p.p0 + j1 + 1;
    const int c0 = split * a.chunk, c1 = min(kv_end, c0 + a.chunk);
    if (c0 >= kv_end) return;
    const int n_tiles = (c1 - c0 + kTileKeys - 1) / kTileKeys;
    if (tid == 0) sh.any_odd = 0;
    __syncthreads();
    auto tile_key = [&](int i) LEAP_INLINE { return c0 + kTileKeys * i; };

    if (a.parent) {
        if (wave == kWideWaves - 1) {
            const TreeLane t = tree_lane(a.parent + p.first, p.n, lane);
            sh.sees[lane] = t.sees;
            const uint64_t bad = __builtin_amdgcn_ballot_w64(t.bad);
            if (lane == 0) sh.bad = bad;
        }
        __syncthreads();
    }
    auto place_of = [&](int j) LEAP_INLINE { return p.p0 + (a.parent ? (int)__popcll(sh.sees[j]) - 1 : j); };

    // ---- the cache's rows ----
    const int kv_dim = a.n_kv_heads * HD;
    const uint32_t row_bytes = (uint32_t)kv_dim * (Q8 ? 1 : 4), head_off = (uint32_t)kvh * HD * (Q8 ? 1 : 4);
    const size_t base = (size_t)p.seq * a.seq_stride;
    const uint32_t bytes = (uint32_t)c1 * row_bytes;  // (rows from there on read as zero)
    const auto rows_r = Q8 ? make_rsrc((brings_v ? a.v8 : a.k8) + base, bytes)
                           : make_rsrc((brings_v ? a.v_cache : a.k_cache) + base, bytes);
    const size_t sbase = (size_t)p.seq * a.scale_stride + (size_t)kvh * a.scale_rows;
    const auto ksr = make_rsrc(Q8 ? a.ks + sbase : nullptr, Q8 ? (uint32_t)c1 * 4u : 0u);
    const auto vsr = make_rsrc(Q8 ? a.vs + sbase : nullptr, Q8 ? (uint32_t)c1 * 4u : 0u);
    // A wave's share of a tile, as it comes from memory.
    //   K, fp32: quads w and w + 4; lane: position lane / 16 of each, C / 2 dims
    //   V, fp32: the same quads; lane: dims lane (and lane + 64), 4 positions
    //   K, 8 bits: positions 8 w + lane / 8, HD / 8 dims (bytes)
    //   V, 8 bits: quad w + 4 (lane / 32) (head_dim 64: 4 w + lane / 16, w < 2), dims 4 (lane % (HD / 4)), 4 positions
    constexpr int RAW = Q8 ? 4 : HD / 8;
    float raw[RAW], sck = 0.0f, scv = 0.0f;
    float sv4[4];
    const int v8_quad = HD == 128 ? w + 4 * (lane >> 5) : 4 * w + (lane >> 4), v8_dim = 4 * (lane & (LR - 1));
    // (the lane's part of an offset into a tile; a tile's rows add a uniform one)
    const uint32_t lane_off = head_off + (Q8 ? (brings_v ? 4u * v8_quad * row_bytes + v8_dim : (8u * w + (lane >> 3)) * row_bytes + (HD / 8) * (lane & 7))
                                             : (brings_v ? 4u * lane : (lane >> 4) * row_bytes + (HD / 4) * (lane & 15)));
    auto load_tile = [&](auto role, int i) LEAP_INLINE {
        constexpr bool V = decltype(role)::value;
        if (i >= n_tiles) return;
        const uint32_t at = (uint32_t)tile_key(i) * row_bytes + lane_off;
        if constexpr (!Q8) {
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const uint32_t quad = 4u * (w + 4 * t) * row_bytes;
                if constexpr (!V) {
#pragma unroll
                    for (int u = 0; u < HD / 64; u++) {
                        const float4 x = buf_load4(rows_r, at + quad + 16 * u);
                        raw[(HD / 16) * t + 4 * u] = x.x;
                        raw[(HD / 16) * t + 4 * u + 1] = x.y;
                        raw[(HD / 16) * t + 4 * u + 2] = x.z;
                        raw[(HD / 16) * t + 4 * u + 3] = x.w;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int u = 0; u < HD / 64; u++)
                            raw[(HD / 16) * t + 4 * u + j] = __int_as_float(
                                __builtin_amdgcn_raw_buffer_load_b32(rows_r, (int)(at + (quad + j * row_bytes) + 256 * u), 0, 0));
                }
            }
        } else if constexpr (!V) {
            if constexpr (HD == 128) {
                const float4 x = buf_load4(rows_r, at);
                raw[0] = x.x;
                raw[1] = x.y;
                raw[2] = x.z;
                raw[3] = x.w;
            } else {
                const float2 x = buf_load2(rows_r, at);
                raw[0] = x.x;
                raw[1] = x.y;
            }
            const int row4 = 4 * (tile_key(i) + 8 * w + (lane >> 3));
            sck = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(ksr, row4, 0, 0));
            scv = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(vsr, row4, 0, 0));
        } else if (HD == 128 || w < 2) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                raw[j] = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(rows_r, (int)(at + j * row_bytes), 0, 0));
            const float4 x = buf_load4(vsr, 4u * (tile_key(i) + 4 * v8_quad));
            sv4[0] = x.x;
            sv4[1] = x.y;
            sv4[2] = x.z;
            sv4[3] = x.w;
        }
    };
    // That share into LDS, split, with its factors.
    auto v_piece = [&](int d, int piece) LEAP_INLINE { return d * 4 + (piece ^ (((d >> 1) ^ (d >> 3)) & 3)); };
    // First looked over, in the vector phase, then split, between the products
    // of the matrix phase (whose waits that fills).
    constexpr int N = HD / 16;  // fp32: a lane's elements of a quad
    constexpr int kPieces = Q8 ? 1 : N;
    float stage_sc[2];
    auto stage_look = [&](auto role, int i) LEAP_INLINE {
        constexpr bool V = decltype(role)::value;
        if (Q8 || i >= n_tiles) return;
        int oddbits = 0, ln = lane;
        asm volatile("" : "+v"(ln));  // (addresses formed anew, for the registers' sake)
        if constexpr (!Q8) {
#pragma unroll
            for (int t = 0; t < 2; t++) {
                float *x = raw + N * t;
                const int quad = w + 4 * t;
                // the lane's largest by position (K: of its one), the quad's;
                // and whether a position stays far below the quad
                constexpr int Y = V ? 4 : 1;
                float y[Y];
                unsigned most;
                bool unlike;
                auto look = [&]() LEAP_INLINE {
                    float all = 0.0f;
#pragma unroll
                    for (int j = 0; j < Y; j++) {
                        y[j] = 0.0f;
#pragma unroll
                        for (int e = j; e < N; e += Y) y[j] = max_abs(y[j], x[e]);
                        all = max_abs(all, y[j]);
                    }
                    const unsigned z = dpp_max16(__float_as_uint(all));
                    const unsigned p0 = __builtin_amdgcn_readlane(z, 0), p1 = __builtin_amdgcn_readlane(z, 16);
                    const unsigned p2 = __builtin_amdgcn_readlane(z, 32), p3 = __builtin_amdgcn_readlane(z, 48);
                    most = max(max(p0, p1), max(p2, p3));
                    const unsigned low = most >= (kUnlike << 23) ? most - (kUnlike << 23) : 0u;
                    if constexpr (V) {
                        unlike = false;
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            unlike |= __builtin_amdgcn_ballot_w64(__float_as_uint(y[j]) >= low) == 0;
                    } else {
                        unlike = min(min(p0, p1), min(p2, p3)) < low;
                    }
                };
                look();
                if (__builtin_expect(!finite_bits(most), 0)) {
                    // zeros in their place, and their positions noted
                    int bits = 0;
#pragma unroll
                    for (int e = 0; e < N; e++)
                        if (!finite_bits(abs_bits(x[e]))) {
                            x[e] = 0.0f;
                            bits |= V ? 1 << (e & 3) : 1 << (ln >> 4);
                        }
#pragma unroll
                    for (int b = 0; b < 4; b++)
                        if (__builtin_amdgcn_ballot_w64((bits >> b) & 1)) oddbits |= 1 << (4 * t + b);
                    look();
                }
                const int e = tile_exp(most);
                stage_sc[t] = exp2_int(13 - e);
                // (every lane writes the same: no branch)
                (V ? sh.vquad : sh.kquad)[i & 3][quad & 1][quad >> 1] = exp2_int(e - 13);
                if (__builtin_expect(unlike, 0)) {
                    // positions far below their neighbours: each by its own exponent
#pragma unroll
                    for (int j = 0; j < Y; j++) {
                        const unsigned top = V ? wave_max_bits(__float_as_uint(y[j])) : dpp_max16(__float_as_uint(y[j]));
                        const int own = top == 0 ? e : tile_exp(top);
#pragma unroll
                        for (int u = j; u < N; u += Y) x[u] = __builtin_amdgcn_ldexpf(x[u], e - own);
                        (V ? sh.vfac : sh.kfac)[i & 3][quad & 1][4 * (quad >> 1) + (V ? j : ln >> 4)] = exp2_int(own - 13);
                    }
                    oddbits |= 256 << t;
                }
            }
        }
        sh.odd[i & 3][wave] = oddbits;
        if (__builtin_expect(oddbits != 0, 0)) sh.any_odd = 1;
    };
    unsigned hi[2], lo[2];
    constexpr int P = WideShared<HD, Q8>::P;
    // (fp32: the lane's first place; the others are 16 positions of K on, 64
    // dims of V on, or in the piece 2 away, where the swizzles repeat)
    auto stage_place = [&](auto role) LEAP_INLINE {
        constexpr bool V = decltype(role)::value;
        int ln = lane;
        asm volatile("" : "+v"(ln));
        const int pos = 4 * w + (ln >> 4);
        return V ? 2 * v_piece(ln, w & 1) + (w >> 1)
                 : 2 * (pos * C + ((HD == 128 ? ln & 15 : (ln & 15) >> 1) ^ (pos & (C - 1)))) + (HD == 128 ? 0 : ln & 1);
    };
    // (a tile past the chunk's last goes where none is read any more)
    auto stage_piece = [&](auto role, int i, int piece, int place) LEAP_INLINE {
        constexpr bool V = decltype(role)::value;
        if constexpr (!Q8) {
            const int t = piece / (N / 2), e2 = piece % (N / 2), h = e2 & 1;
            split2_scaled(raw[N * t + 2 * e2], raw[N * t + 2 * e2 + 1], stage_sc[t], hi[h], lo[h]);
            if (h == 0) return;
            const int at = V ? (t ? place ^ 4 : place) + 2 * 4 * 64 * (e2 >> 1) : place + 2 * 16 * C * t + (e2 >> 1);
            u32x2 *to_h = reinterpret_cast<u32x2 *>(V ? sh.v[i % 3][0] : sh.k[i & 1][0]);
            u32x2 *to_l = reinterpret_cast<u32x2 *>(V ? sh.v[i % 3][P - 1] : sh.k[i & 1][P - 1]);
            to_h[at] = u32x2{hi[0], hi[1]};
            to_l[at] = u32x2{lo[0], lo[1]};
        } else {
            int ln = lane;
            asm volatile("" : "+v"(ln));
            if constexpr (!V) {
                const int pos = 8 * w + (ln >> 3);
                if constexpr (HD == 128) {
#pragma unroll
                    for (int u = 0; u < 2; u++)
                        sh.k[i & 1][0][pos * C + ((2 * (ln & 7) + u) ^ (pos & (C - 1)))] =
                            bytes_half8(__float_as_uint(raw[2 * u]), __float_as_uint(raw[2 * u + 1]));
                } else {
                    sh.k[i & 1][0][pos * C + ((ln & 7) ^ (pos & (C - 1)))] =
                        bytes_half8(__float_as_uint(raw[0]), __float_as_uint(raw[1]));
                }
                if ((ln & 7) == 0) sh.kfac[i & 3][(pos >> 2) & 1][4 * (pos >> 3) + (pos & 3)] = sck + 0.0f * scv;
            } else if (HD == 128 || w < 2) {
                int quad = v8_quad, d0 = v8_dim;
                asm volatile("" : "+v"(quad), "+v"(d0));  // (addresses formed anew, as below)
                const int piece = 2 * (quad >> 2) + (quad & 1), half = (quad >> 1) & 1;
                unsigned x[4];
#pragma unroll
                for (int j = 0; j < 4; j++) x[j] = __float_as_uint(raw[j]) ^ 0x80808080u;
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const unsigned sel = 0x0c000c00u | (unsigned)(4 + c) << 16 | (unsigned)c;
                    const half2v p0 = bytes_half(__builtin_amdgcn_perm(x[1], x[0], sel) | 0x64006400u);
                    const half2v p1 = bytes_half(__builtin_amdgcn_perm(x[3], x[2], sel) | 0x64006400u);
                    const int d = d0 + c;
                    *(reinterpret_cast<u32x2 *>(&sh.v[i % 3][0][v_piece(d, piece)]) + half) =
                        u32x2{__builtin_bit_cast(unsigned, p0), __builtin_bit_cast(unsigned, p1)};
                }
                if ((ln & (LR - 1)) == 0)
#pragma unroll
                    for (int j = 0; j < 4; j++) sh.vfac[i & 3][quad & 1][4 * (quad >> 1) + j] = sv4[j];
            }
        }
    };
    auto stage_tile = [&](auto role, int i) LEAP_INLINE {
        stage_look(role, i);
#pragma unroll
        for (int x = 0; x < kPieces; x++) stage_piece(role, i, x, stage_place(role));
    };

    // ---- Q: 32 rows a wave, in registers as the products' B operand ----
    // K's first two tiles and V's first are on their way meanwhile, if this
    // call does not bring rows of them; the chunk's new rows go to the cache
    // first (by every workgroup that reads them, the same bytes).
    const int t0 = a.fused ? max(c0 - p.p0, 0) : 0, n_new = a.fused ? max(min(c1 - p.p0, p.n) - t0, 0) : 0;
    const bool early = n_new == 0 || c0 + 2 * kTileKeys <= p.p0;
    auto by_role = [&](auto f) LEAP_INLINE {
        if (brings_v)
            f(std::true_type{});
        else
            f(std::false_type{});
    };
    if (early) by_role([&](auto role) LEAP_INLINE { load_tile(role, 0); });
    for (int i = tid / LR; i < 2 * n_new; i += kWideThreads / LR) {
        const bool value = i >= n_new;
        const int j = t0 + (value ? i - n_new : i), lr = tid & (LR - 1);
        float4 y = reinterpret_cast<const float4 *>(value ? a.v_new : a.k_new)[((size_t)(p.first + j) * a.n_kv_heads + kvh) * LR + lr];
        if (!value) y = rope4(y, a.rope[(size_t)place_of(j) * LR + lr]);
        float f = 0.0f;
        const int q = Q8 ? quantize_row<HD>(y, &f) : 0;
        store_row<HD, Q8>(a, p.seq, p.p0 + j, kvh * LR + lr, y, q, f, value);
    }
    constexpr int QL = WideShared<HD, Q8>::kQLow, QR = KS - QL;  // low halves of Q in LDS, in registers
    const bool idle = r0 + 32 * wave >= rows;  // no rows: this wave only brings its share
    // Rows of q and out are read and written whole, LR lanes a row, and turned
    // through LDS; all waves take turns with the tile's rows of q.
    constexpr int RW = kWave / LR, kAhead = 8;
    const int lr = lane & (LR - 1), sub = lane / LR;
    auto row_at = [&](int r, int *j) LEAP_INLINE {
        *j = (int)fast_div((uint32_t)r, a.by_group);
        return ((size_t)(p.first + *j) * a.n_heads + kvh * a.group + r - *j * a.group) * LR + lr;
    };
    {
        const int n_rows = (min(BM, rows - r0) + 31) & ~31;
        for (int b = RW * wave + sub; b < n_rows; b += RW * kWideWaves * kAhead) {
            float4 x[kAhead], turn[kAhead];
            int j[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; i++) {
                const int r = min(r0 + b + RW * kWideWaves * i, rows - 1);
                x[i] = reinterpret_cast<const float4 *>(a.q)[row_at(r, &j[i])];
                turn[i] = a.rope[(size_t)place_of(j[i]) * LR + lr];
            }
#pragma unroll
            for (int i = 0; i < kAhead; i++) {
                const int row = b + RW * kWideWaves * i;
                if (row >= n_rows) break;
                const float4 y = rope4(x[i], turn[i]);
                unsigned mx = dpp_max16(max4_bits(0u, y));
                if constexpr (HD == 128) mx = max(mx, (unsigned)__shfl_xor((int)mx, 16));
                const bool good = finite_bits(mx) && !(a.parent && (sh.bad >> j[i] & 1));
                const int e = tile_exp(good ? mx : 0u);
                const float sc = good ? exp2_int(13 - e) : 0.0f;
                half2v h[2], l[2];
                split2(y.x * sc, y.y * sc, h[0], l[0]);
                split2(y.z * sc, y.w * sc, h[1], l[1]);
                const int at = (row & 31) * C + ((lr >> 1) ^ (row & (C - 1)));
                *(reinterpret_cast<u32x2 *>(&sh.q[row >> 5][0][at]) + (lr & 1)) =
                    u32x2{__builtin_bit_cast(unsigned, h[0]), __builtin_bit_cast(unsigned, h[1])};
                *(reinterpret_cast<u32x2 *>(&sh.q[row >> 5][1][at]) + (lr & 1)) =
                    u32x2{__builtin_bit_cast(unsigned, l[0]), __builtin_bit_cast(unsigned, l[1])};
                if (lr == 0) sh.qf[row >> 5][row & 31] = good ? exp2_int(e - 13) * a.scale_log2 : __uint_as_float(0x7fc00000u);
            }
        }
    }
    if (n_new) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (n_new) __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");  // (L1 may hold parts of the new rows' lines)
    half8v qh[KS], ql[KS];
#pragma unroll
    for (int t = 0; t < KS; t++) {
        const int at = n * C + ((2 * t + g) ^ (n & (C - 1)));
        qh[t] = sh.q[wave][0][at];
        ql[t] = sh.q[wave][1][at];
    }
    const float qf = sh.qf[wave][n];
    __syncthreads();
#pragma unroll
    for (int t = QR; t < KS; t++) sh.ql[wave][t - QR][lane] = ql[t];

    const int all_see = a.parent ? p.p0 - 1 : p.p0 + j0;  // the last position that every row of the tile sees
    f32x16 o[VB], s;
#pragma unroll
    for (int v = 0; v < VB; v++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[v][r] = 0.0f;
    half8v ph[2], pl[2];
    float ref = kNothing, sum = 0.0f, vrun = 1.0f;  // (vrun: O's unit in the lane's row)

    // (a lane's pieces: K piece 2 t + g of position n, V piece 2 u + g of dim
    // 32 v + n; the swizzles leave t and u as an exclusive or on the first's
    // index.  Formed anew in each phase: kept, they would take 16 registers.)
    const int k_first = n * C + (g ^ (n & (C - 1))), v_first = v_piece(n, g);
    auto clear_scores = [&]() LEAP_INLINE {
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = 0.0f;
    };
    auto scores = [&](int i) LEAP_INLINE {
        clear_scores();
        const half8v *k = sh.k[i & 1][0];
        int kf = k_first;
        asm volatile("" : "+v"(kf));
#pragma unroll
        for (int t = 0; t < KS; t++) {
            const int at = kf ^ (2 * t);
            const half8v kh = k[at];
            s = mfma32(kh, t < QR ? ql[t < QR ? t : 0] : sh.ql[wave][t < QR ? 0 : t - QR][lane], s);
            if constexpr (!Q8) s = mfma32(k[at + 32 * C], qh[t], s);
            s = mfma32(kh, qh[t], s);
        }
    };
    // The scores of tile i + 1 and the weighted values of tile i, in turns: a
    // product that adds to the one before it would wait for it.  (After the
    // last tile the scores are of what an earlier one left, and not used.)
    auto matrix = [&](auto role, int i, int next) LEAP_INLINE {
        clear_scores();
        int kf = k_first, vf = v_first;
        asm volatile("" : "+v"(kf), "+v"(vf));
        const int place = Q8 ? 0 : stage_place(role);
        const half8v *k = sh.k[(i + 1) & 1][0], *x = sh.v[i % 3][0];
        constexpr int D = 2;  // steps that the operands are read ahead
        half8v kh[D + 1], kl[D + 1], vh[D + 1], vl[D + 1], low[D + 1];
        auto read = [&](int t) LEAP_INLINE {
            const int ka = kf ^ (2 * t), va = (vf ^ (2 * (t / VB))) + 128 * (t % VB), e = t % (D + 1);
            kh[e] = k[ka];
            if constexpr (!Q8) kl[e] = k[ka + 32 * C];
            low[e] = t < QR ? ql[t < QR ? t : 0] : sh.ql[wave][t < QR ? 0 : t - QR][lane];
            vh[e] = x[va];
            if constexpr (!Q8) vl[e] = x[va + 4 * HD];
        };
#pragma unroll
        for (int t = 0; t < D; t++) read(t);
#pragma unroll
        for (int t = 0; t < KS; t++) {
            const int u = t / VB, v = t % VB, e = t % (D + 1);
            if (t + D < KS) read(t + D);
            __builtin_amdgcn_sched_barrier(0);
            s = mfma32(kh[e], qh[t], s);
            o[v] = mfma32(vh[e], pl[u], o[v]);
            __builtin_amdgcn_sched_barrier(0);
            if (Q8 ? t == 1 : t < kPieces) stage_piece(role, next, Q8 ? 0 : t, place);
            if constexpr (!Q8) {
                s = mfma32(kl[e], qh[t], s);
                o[v] = mfma32(vl[e], ph[u], o[v]);
                __builtin_amdgcn_sched_barrier(0);
            }
            s = mfma32(kh[e], low[e], s);
            o[v] = mfma32(vh[e], ph[u], o[v]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // fp32: s times the factors of a tile that may have unlike quads, times f
    // (quad 2 t + half of the tile came with wave quad % 4)
    auto by_factors = [&](auto role, int i, int half, f32x16 &s, float f) LEAP_INLINE {
        constexpr bool V = decltype(role)::value;
        const int *bits = &sh.odd[i & 3][V ? half : 4 + half];
        const float *own = (V ? sh.vfac : sh.kfac)[i & 3][half], *all = (V ? sh.vquad : sh.kquad)[i & 3][half];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const bool unlike = (bits[2 * (t & 1)] >> (8 + (t >> 1))) & 1;
            const float4 x = *reinterpret_cast<const float4 *>(own + 4 * t);
            const float y = all[t];
            s[4 * t] *= (unlike ? x.x : y) * f;
            s[4 * t + 1] *= (unlike ? x.y : y) * f;
            s[4 * t + 2] *= (unlike ? x.z : y) * f;
            s[4 * t + 3] *= (unlike ? x.w : y) * f;
        }
    };
    auto softmax = [&](int i) LEAP_INLINE {
        constexpr int F = Q8 ? 16 : 4, P = 16 / F;  // factors of a lane, scores of each
        const int key0 = tile_key(i);
        const float *kfs = Q8 ? sh.kfac[i & 3][g] : sh.kquad[i & 3][g], *vfs = Q8 ? sh.vfac[i & 3][g] : sh.vquad[i & 3][g];
        // scores are s[r] kf[r / P] (8 bits: s[r]); the factors are positive (or NaN in a row without result)
        float kf[F];
#pragma unroll
        for (int t = 0; t < F; t++) kf[t] = kfs[t] * qf;
        if constexpr (Q8) {
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] *= kf[r];
        }
        int odd = 0;
        if (!Q8 && __builtin_expect(__builtin_amdgcn_readfirstlane(sh.any_odd), 0)) {
#pragma unroll
            for (int x = 0; x < kWideWaves; x++) odd |= sh.odd[i & 3][x];
            odd = __builtin_amdgcn_readfirstlane(odd);
        }
        if (!Q8 && __builtin_expect(odd, 0)) {
            int half = lane;
            asm volatile("" : "+v"(half));  // (formed anew, for the registers' sake, here and below)
            half >>= 5;
            // each position by its own factor, and not by one that a position
            // the row does not see has a part in: that may be infinite
            by_factors(std::false_type{}, i, half, s, qf);
#pragma unroll
            for (int t = 0; t < F; t++) kf[t] = 1.0f;
            if (__builtin_expect(odd & 255, 0))
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int quad = 2 * (r >> 2) + half;  // waves quad & 3 brought it, V and K
                    const int both = sh.odd[i & 3][quad & 3] | sh.odd[i & 3][4 + (quad & 3)];
                    if ((both >> (4 * (quad >> 2) + (r & 3))) & 1) s[r] = __uint_as_float(0x7fc00000u);
                }
        }
        if (__builtin_expect(key0 + kTileKeys > c1 || key0 + kTileKeys - 1 > all_see, 0)) {
            // visible: positions up to `limit`, and of a tree's nodes those of `sees`
            int ln = lane;
            asm volatile("" : "+v"(ln));  // (formed anew, for the registers' sake)
            const int my_j = (int)fast_div((uint32_t)min(r0 + 32 * wave + (ln & 31), rows - 1), a.by_group);
            const int first = key0 + 4 * (ln >> 5);
            int limit = p.p0 + my_j;
            uint64_t sees = 0;
            if (a.parent) {
                limit = p.p0 - 1;
                sees = sh.sees[my_j];
            }
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int key = first + 8 * (r >> 2) + (r & 3);
                const bool see = key <= limit || ((sees >> ((key - p.p0) & 63)) & 1);
                if (!see || key >= c1) s[r] = -__builtin_inff();
            }
            if constexpr (!Q8)
#pragma unroll
                for (int t = 0; t < F; t++) kf[t] = kf[t] == 0.0f ? 1e-38f : kf[t];  // (an underflown factor times -inf)
        }
        float mt = -__builtin_inff();
        if constexpr (!Q8) {
#pragma unroll
            for (int t = 0; t < F; t++)
                mt = fmaxf(mt, kf[t] * fmaxf(fmaxf(s[4 * t], s[4 * t + 1]), fmaxf(s[4 * t + 2], s[4 * t + 3])));
        } else {
#pragma unroll
            for (int r = 0; r < 16; r++) mt = fmaxf(mt, s[r]);
        }
        // (the reference and O's unit move as in many_attention.hpp: most
        // tiles leave both, and need no maximum over both lanes of a row)
        auto inverse = [](float x) LEAP_INLINE { return __uint_as_float(0x7f000000u - __float_as_uint(x)); };  // (of powers of two)
        const float vinv = inverse(vrun);
        float most = vfs[0];
#pragma unroll
        for (int t = 1; t < F; t++) most = fmaxf(most, vfs[t]);
        if constexpr (Q8) asm volatile("" ::: "memory");  // (sixteen factors are read again rather than kept)
        Half8 h[2], l[2];
        auto split = [&](int r, float x, float y, float f, float g) LEAP_INLINE {
            split2_by(x, y, f, g, h[r >> 3].h[(r & 7) / 2], l[r >> 3].h[(r & 7) / 2]);
        };
        auto prob = [&](int r, float off) LEAP_INLINE { return fast_exp2(Q8 ? s[r] - off : __builtin_fmaf(s[r], kf[r / P], -off)); };
        // (scales of 8 bits are no powers of two: the next)
        const bool fits = __builtin_amdgcn_ballot_w64(!fits_unit(mt, ref, (Q8 ? 2.0f : 1.0f) * most * vinv)) == 0;
        float total = sum;
        {
            const float off = ref - kProbBias;
            float vf[F];  // (0 for a scale of NaN, which a masked probability may meet)
#pragma unroll
            for (int t = 0; t < F; t++) vf[t] = Q8 ? fmaxf(vfs[t] * vinv, 0.0f) : vfs[t] * vinv;
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float x = prob(r, off), y = prob(r + 1, off);
                total += x + y;
                split(r, x, y, vf[r / P], vf[(r + 1) / P]);
            }
        }
        if (__builtin_expect(!fits || odd, 0)) {
            // all of that again
            mt = half_max(mt);
            const float now = mt > ref + kProbRoom ? ceilf(mt) : ref, up = now - ref, off = now - kProbBias;
            ref = now;
            total = sum * fast_exp2(-up);
#pragma unroll
            for (int r = 0; r < 16; r++) {
                s[r] = prob(r, off);
                total += s[r];
            }
            int half = lane;
            asm volatile("" : "+v"(half)::"memory");
            half >>= 5;
            if constexpr (Q8) {
#pragma unroll
                for (int r = 0; r < 16; r++) s[r] *= fmaxf(sh.vfac[i & 3][half][r], 0.0f) * exp2_int(-kRoom);
            } else if (odd) {
                by_factors(std::true_type{}, i, half, s, exp2_int(-kRoom));
            } else {
#pragma unroll
                for (int r = 0; r < 16; r++) s[r] *= sh.vquad[i & 3][half][r >> 2] * exp2_int(-kRoom);
            }
            float top = fmaxf(s[0], s[1]);
#pragma unroll
            for (int r = 2; r < 16; r += 2) top = fmaxf(fmaxf(top, s[r]), s[r + 1]);
            const int was = (int)(__float_as_uint(vrun) >> 23) - 127, unit = next_unit(was, half_max(top), up);
            const float os = fast_exp2((float)(was - unit) - up), by = exp2_int(kRoom - unit);
            vrun = exp2_int(unit);
            if (__builtin_amdgcn_ballot_w64(os != 1.0f))
#pragma unroll
                for (int v = 0; v < VB; v++) o[v] *= os;
#pragma unroll
            for (int r = 0; r < 16; r += 2) split(r, s[r], s[r + 1], by, by);
        }
        sum = total;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            ph[u] = h[u].v;
            pl[u] = l[u].v;
        }
    };

    // ---- the half-steps ----
    by_role([&](auto role) LEAP_INLINE {
        constexpr bool V = decltype(role)::value;
        if (!early) load_tile(role, 0);
        stage_tile(role, 0);
        load_tile(role, 1);
        if constexpr (!V) {
            stage_tile(role, 1);
            load_tile(role, 2);
        }
        __syncthreads();
        if constexpr (!V) __syncthreads();
        if (!idle) scores(0);
        __syncthreads();
        for (int i = 0; i < n_tiles; i++) {
            const int next = V ? i + 1 : i + 2;
            if (!idle) softmax(i);
            __builtin_amdgcn_sched_barrier(0);
            stage_look(role, next);
            __syncthreads();
            if (!idle) {
                __builtin_amdgcn_s_setprio(1);  // (the matrix phase's few instructions before the vector phase's many)
                matrix(role, i, next);
                __builtin_amdgcn_s_setprio(0);
            } else {
#pragma unroll
                for (int x = 0; x < kPieces; x++) stage_piece(role, next, x, stage_place(role));
            }
            load_tile(role, next + 1);
            __syncthreads();
        }
        if constexpr (V) __syncthreads();
    });
    if (idle) return;

    // ---- results: register r of block v is dim 32 v + 8 (r / 4) + 4 g + r % 4 ----
    sum += __shfl_xor(sum, 32);
    const bool none = sum == 0.0f;  // (a chunk none of whose positions the row sees)
    const float inv = none ? 0.0f : vrun / sum;
    float4 *rows_o = sh.o[wave];
#pragma unroll
    for (int v = 0; v < VB; v++)
#pragma unroll
        for (int t = 0; t < 4; t++)
            rows_o[n * LR + ((8 * v + 2 * t + g) ^ (n & (LR - 1)))] =
                make_float4(o[v][4 * t] * inv, o[v][4 * t + 1] * inv, o[v][4 * t + 2] * inv, o[v][4 * t + 3] * inv);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (this wave's own rows)
    __builtin_amdgcn_wave_barrier();
    const int n_split = a.spread ? (kv_end + a.chunk - 1) / a.chunk : 1;
    const size_t rec = ((size_t)group_i * a.splits + split) * BM + 32 * wave;
    for (int b = 0; b < 32; b += RW) {
        const int row = b + sub, r = r0 + 32 * wave + row;
        if (r >= rows) break;
        const float4 x = rows_o[row * LR + (lr ^ (row & (LR - 1)))];
        int j;
        if (n_split == 1)
            reinterpret_cast<float4 *>(a.out)[row_at(r, &j)] = x;
        else
            reinterpret_cast<float4 *>(a.ws_o)[(rec + row) * LR + lr] = x;
    }
    if (n_split > 1 && g == 0 && r0 + 32 * wave + n < rows)
        a.ws_lse[rec + n] = none ? -__builtin_inff() : ref + log2f(sum) - kProbBias;
}

}  // namespace leap

#undef LEAP_INLINE
