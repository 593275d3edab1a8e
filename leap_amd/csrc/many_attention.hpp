// Attention of several new tokens of each sequence over its cache (prompts,
// trees of drafted tokens), and of any number of them over an 8-bit cache.
//
// For the q heads that share a KV head, the (token, head) pairs of a
// sequence are the rows r = token * group + head of one product: tiles of
// 16 rows of Q (wide_attention.hpp: of 256) against the cache's rows, so that
// a K or V row is read once for all of a tile's rows.  A workgroup takes one
// tile and one chunk of positions; its waves, four or (8 bits, whose rows are
// a quarter of the bytes) eight, take 32 positions each in turn and keep an
// online softmax of their own, combined at the end.  Chunks of one tile leave
// records (output, log2 of the sum) that the last one to arrive adds up.
//
// Products.  S^T = K Q^T and O^T = V^T P^T as 16x16x32 MFMAs in fp16, with a
// lane holding one row of Q throughout: S^T's column is the lane's row, its
// four registers per block are positions 4 (lane / 16) + i, and with the
// contraction over positions taken in that same order (slot (g, 4 b + i) is
// position 16 b + 4 g + i) those registers are O^T's B operand as they are.
// No score leaves its lane.
//
// fp32 operands in fp16 products: x = 2^e (h + l), h = fp16(x 2^-e) and
// l = fp16(x 2^-e - h), both rounded to nearest, with e such that the
// largest of x's row is in [2^13, 2^14) (wide_attention.hpp: of a quad of
// rows, where these are within 2^4 of each other).  h and l together hold x to
// 2^-22 of itself, or to 2^-38 of the row's largest (quads: 2^-34), half of
// fp16's least step, whichever is more; rows below 2^-100 to 2^-138.
// h h' + h l' + l h' leaves out l l' < 2^-22 |x x'|, of either
// sign: on sums of 128 terms and more that is fp32's own error.  Three fp16
// MFMAs take 3/16 of the time of the fp32 MFMAs of the product.  The
// probabilities are split the same way, with 2^7 folded into their exponent
// and each value row's 2^e into them, over a power of two that follows the
// largest such product that the row of Q has met (next_unit): its weighted
// values are held to 2^-22 of themselves, or 2^-30 of the largest.  8-bit
// values are exact in fp16 and take two products.
//
// Rows with infinities or NaN: such a key or value makes NaN of the output
// rows that see it, and of those only: its elements are replaced by zero in
// the products and its scores by NaN where they are not masked.
#pragma once

#include "decode_attention.hpp"

namespace leap {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));

constexpr int kAppendWaves = 4;                        // waves of a workgroup of the append kernel
constexpr int kTileKeys = 32;                          // positions a wave takes at a time
constexpr int kManySplits = 64;                        // chunks of a tile, at most
constexpr int kTreeMax = 64;                           // nodes of a sequence's tree
constexpr float kProbBias = 7.0f, kProbRoom = 8.0f;    // probabilities are 2^(score - reference + 7) <= 2^15
constexpr int kLeastUnit = -110;                       // the least exponent of O's unit
constexpr float kNothing = -3.4028234664e38f;          // the softmax reference of a row that has seen nothing
constexpr int kRoom = 16;                              // 2^16: probabilities times factors over that are finite
constexpr float kAmaxFloor = 7.888609052210118e-31f;   // 2^-100: the least largest magnitude of an 8-bit head row

// One launch over one layer.  begin NULL: one token a sequence, row i of
// sequence i (then pos NULL: position pos_scalar).
struct ManyArgs {
    const float *q, *k_new, *v_new;  // rows of [n_heads*HD], [n_kv_heads*HD]
    float *out;
    float *k_cache, *v_cache;        // fp32 cache: sequence 0's rows of this layer
    int8_t *k8, *v8;                 // 8-bit cache: the same, values
    float *ks, *vs;                  // and scales, [n_kv_heads][scale_rows]
    const float4 *rope;
    const int *begin, *pos, *parent;
    float *ws_o, *ws_lse;            // records of split tiles: [group][split][rows][HD], [group][split][rows]
    int *counters;                   // [group], zero between launches
    long long seq_stride;            // elements between sequences
    long long scale_stride;          // floats between sequences
    int scale_rows;
    int n_seq, n_tokens, max_tokens, max_pos, pos_scalar;
    int n_heads, n_kv_heads, group;
    int slots;                       // tiles of all sequences, at most
    int chunk, splits;               // positions of a chunk, chunks of the longest sequence
    int fused;                       // the attention kernel stores the new rows itself (else many_append_kernel ran)
    int spread;                      // a tile's chunks lie on all XCDs, and many_merge_kernel adds up their records
    float scale_log2;
    FastDiv by_group, by_kv_heads, by_splits;
};

__device__ __forceinline__ int wave_scan_add(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);  // row_shr:2
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);  // row_shr:4
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);  // row_shr:8
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31
    return v;
}

// Lane i's sequence base + i of the packed batch: its first token row, its
// tokens (0 where there is none) and its first position.  A sequence is
// skipped (n = -1) where its rows leave [0, n_tokens), where it has more than
// max_tokens tokens or positions outside [0, max_pos], and from one whose rows
// go backwards on.  *stop: the sequences behind these are skipped too.
struct SeqLane {
    int first, n, p0;
};
__device__ __forceinline__ SeqLane seq_lane(const ManyArgs &a, int base, int lane, bool *stop)
{
    const int i = base + lane;
    SeqLane s{0, 0, 0};
    bool back = false;
    if (i < a.n_seq) {
        s.first = a.begin[i];
        const int end = a.begin[i + 1];
        s.p0 = a.pos[i];
        back = end < s.first;
        s.n = s.first >= 0 && end <= a.n_tokens ? end - s.first : -1;
    }
    const uint64_t backs = __builtin_amdgcn_ballot_w64(back);
    *stop = backs != 0;
    if (backs && lane >= __builtin_ctzll(backs)) s.n = i < a.n_seq ? -1 : 0;
    if (s.n > 0 && (s.n > a.max_tokens || s.p0 < 0 || s.p0 > a.max_pos + 1 - s.n)) s.n = -1;
    return s;
}

// The tile `slot` of the batch (tiles of BM rows, a sequence's last first:
// with causal masks they see the most positions): seq < 0 where there is
// none, n < 0 for a skipped sequence's (with begin, those have no tiles).
struct Place {
    int seq, tile, first, n, p0;
};
template <int BM>
__device__ __forceinline__ Place find_place(const ManyArgs &a, int slot, int lane)
{
    Place p{-1, 0, 0, 0, 0};
    if (!a.begin) {
        // (one tile a sequence: group <= 16)
        if (slot >= a.n_seq) return p;
        const int p0 = a.pos ? a.pos[slot] : a.pos_scalar;
        return Place{slot, 0, slot, p0 < 0 || p0 > a.max_pos ? -1 : 1, p0};
    }
    int before = 0;
    bool stop = false;
    for (int base = 0; base < a.n_seq && !stop; base += kWave) {
        const SeqLane s = seq_lane(a, base, lane, &stop);
        const int tiles = s.n > 0 ? (s.n * a.group + BM - 1) / BM : 0;
        const int upto = wave_scan_add(tiles);
        const int total = __builtin_amdgcn_readlane(upto, kWave - 1);
        if (slot - before < total) {
            const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > slot - before));
            p.seq = base + l;
            p.tile = __builtin_amdgcn_readlane(upto, l) - 1 - (slot - before);
            p.first = __builtin_amdgcn_readlane(s.first, l);
            p.n = __builtin_amdgcn_readlane(s.n, l);
            p.p0 = __builtin_amdgcn_readlane(s.p0, l);
            return p;
        }
        before += total;
    }
    return p;
}

// Lane j's node j of a tree of n <= 64 nodes: the bits of its ancestors and
// itself, by six doublings of the steps upwards.  A parent outside [-1, j)
// counts as -1 there, and marks the node and its descendants bad: no results.
struct TreeLane {
    uint64_t sees;
    bool bad;
};
__device__ __forceinline__ TreeLane tree_lane(const int *parent, int n, int lane)
{
    int up = lane < n ? parent[lane] : -1;
    int bad = up < -1 || up >= lane;
    if (bad) up = -1;
    unsigned lo = lane < 32 ? 1u << lane : 0u, hi = lane < 32 ? 0u : 1u << (lane - 32);
    for (int k = 0; k < 6; k++) {
        const int from = max(up, 0);
        const unsigned lo2 = __shfl(lo, from), hi2 = __shfl(hi, from);
        const int up2 = __shfl(up, from), bad2 = __shfl(bad, from);
        if (up >= 0) {
            lo |= lo2;
            hi |= hi2;
            bad |= bad2;
            up = up2;
        }
    }
    return TreeLane{((uint64_t)hi << 32) | lo, bad != 0};
}

__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ bool finite_bits(unsigned b) { return b < 0x7f800000u; }
__device__ __forceinline__ unsigned max4_bits(unsigned m, float4 x)
{
    return max(max(max(m, abs_bits(x.x)), max(abs_bits(x.y), abs_bits(x.z))), abs_bits(x.w));
}
__device__ __forceinline__ unsigned dpp_max16(unsigned x)
{
    // over the 16 lanes of a row, in every lane (row_ror)
    x = max(x, (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0x121, 0xF, 0xF, true));
    x = max(x, (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0x122, 0xF, 0xF, true));
    x = max(x, (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0x124, 0xF, 0xF, true));
    x = max(x, (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0x128, 0xF, 0xF, true));
    return x;
}
__device__ __forceinline__ unsigned wave_max_bits(unsigned x)
{
    x = dpp_max16(x);
    const unsigned a = __builtin_amdgcn_readlane(x, 0), b = __builtin_amdgcn_readlane(x, 16);
    const unsigned c = __builtin_amdgcn_readlane(x, 32), d = __builtin_amdgcn_readlane(x, 48);
    return max(max(a, b), max(c, d));
}

// The exponent that a tile of largest magnitude `bits` is scaled by: in
// [-100, 127], and 2^(13 - e), 2^(e - 13) as floats.
__device__ __forceinline__ int tile_exp(unsigned bits) { return max((int)(bits >> 23), 27) - 127; }
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// x = h + l in fp16, to 2^-22 relative (see above), x already scaled.
__device__ __forceinline__ void split2(float x, float y, half2v &h, half2v &l)
{
    h = half2v{(_Float16)x, (_Float16)y};
    asm("" : "+v"(h));  // (the packed pair is what the remainders are taken from)
    l = half2v{(_Float16)(x - (float)h.x), (_Float16)(y - (float)h.y)};
}
// The same of x * f and y * g, whose products are not rounded first.
__device__ __forceinline__ void split2_by(float x, float y, float f, float g, half2v &h, half2v &l)
{
    h = half2v{(_Float16)(x * f), (_Float16)(y * g)};
    asm("" : "+v"(h));
    l = half2v{(_Float16)__builtin_fmaf(x, f, -(float)h.x), (_Float16)__builtin_fmaf(y, g, -(float)h.y)};
}
union Half8 {
    half8v v;
    half2v h[4];
};
__device__ __forceinline__ float4 mul4(float4 a, float4 b) { return make_float4(a.x * b.x, a.y * b.y, a.z * b.z, a.w * b.w); }
__device__ __forceinline__ void split8(float4 a, float4 b, half8v &hi, half8v &lo)
{
    Half8 h, l;
    split2(a.x, a.y, h.h[0], l.h[0]);
    split2(a.z, a.w, h.h[1], l.h[1]);
    split2(b.x, b.y, h.h[2], l.h[2]);
    split2(b.z, b.w, h.h[3], l.h[3]);
    hi = h.v;
    lo = l.v;
}

// The same of x * sc and y * sc, two fused mixed-precision operations each.
// (What comes out goes to LDS: the compiler knows no hazards of instructions
// it does not see, so these never feed a matrix instruction.)
__device__ __forceinline__ void split2_scaled(float x, float y, float sc, unsigned &h, unsigned &l)
{
    asm("v_fma_mixlo_f16 %0, %1, %2, 0" : "=v"(h) : "v"(x), "s"(sc));
    asm("v_fma_mixhi_f16 %0, %1, %2, 0" : "+v"(h) : "v"(y), "s"(sc));
    asm("v_fma_mixlo_f16 %0, %1, %2, -%3 op_sel_hi:[0,0,1]" : "=v"(l) : "v"(x), "s"(sc), "v"(h));
    asm("v_fma_mixhi_f16 %0, %1, %2, -%3 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "+v"(l) : "v"(y), "s"(sc), "v"(h));
}
// The larger magnitude; NaN if either is.
__device__ __forceinline__ float max_abs(float m, float x) { return __builtin_elementwise_maximum(m, __builtin_fabsf(x)); }

__device__ __forceinline__ float max4_abs(float m, float4 x)
{
    return max_abs(max_abs(max_abs(max_abs(m, x.x), x.y), x.z), x.w);
}

// Infinities and NaN replaced by zero; whether there were any.
__device__ __forceinline__ bool zero_bad(float4 &x)
{
    const bool a = finite_bits(abs_bits(x.x)), b = finite_bits(abs_bits(x.y));
    const bool c = finite_bits(abs_bits(x.z)), d = finite_bits(abs_bits(x.w));
    x = make_float4(a ? x.x : 0.0f, b ? x.y : 0.0f, c ? x.z : 0.0f, d ? x.w : 0.0f);
    return !(a && b && c && d);
}

// int8 values to fp16, exactly: with the sign bit flipped a byte u = x + 128
// placed under 0x64 is the fp16 number 1024 + u.
__device__ __forceinline__ half2v bytes_half(unsigned two)
{
    return __builtin_bit_cast(half2v, two) - half2v{(_Float16)1152.0f, (_Float16)1152.0f};
}
// The same of bytes alone (the halves 0x0000 | byte, subnormals of fp16):
// values times 2^-9, as exact.  (Left subnormal, values cost the products
// bits: errors of 1.7e-6 for 5e-7.)
__device__ __forceinline__ half2v bytes_small(unsigned two)
{
    const _Float16 up = (_Float16)32768.0f, off = (_Float16)-0.25f;
    return __builtin_elementwise_fma(__builtin_bit_cast(half2v, two), half2v{up, up}, half2v{off, off});
}
__device__ __forceinline__ half8v bytes_half8(unsigned a, unsigned b)
{
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    Half8 r;
    r.h[0] = bytes_half(__builtin_amdgcn_perm(0x64646464u, a, 0x04010400u));
    r.h[1] = bytes_half(__builtin_amdgcn_perm(0x64646464u, a, 0x04030402u));
    r.h[2] = bytes_half(__builtin_amdgcn_perm(0x64646464u, b, 0x04010400u));
    r.h[3] = bytes_half(__builtin_amdgcn_perm(0x64646464u, b, 0x04030402u));
    return r.v;
}

__device__ __forceinline__ f32x4 mfma16(half8v a, half8v b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// ---- the rows of the new tokens into the cache -------------------------------

// One head row of HD elements over HD / 4 lanes as int8 values and a scale:
// a = max(largest magnitude, 2^-100), scale a / 127, value rint(x (127 / a)),
// in fp32.  With an infinity or a NaN the scale is NaN, which is what the
// row then stands for.  Every lane returns its four values and the scale.
__device__ __forceinline__ void quantize_scale(unsigned max_bits, float *r, float *scale)
{
    const float a = fmaxf(__uint_as_float(max_bits), kAmaxFloor);
    *r = 127.0f / a;
    *scale = finite_bits(max_bits) ? a / 127.0f : __uint_as_float(0x7fc00000u);
}
__device__ __forceinline__ int quantize4(float4 x, float r)
{
    return ((int)rintf(x.x * r) & 255) | (((int)rintf(x.y * r) & 255) << 8) | (((int)rintf(x.z * r) & 255) << 16) |
           ((int)rintf(x.w * r) << 24);
}
template <int HD>
__device__ __forceinline__ int quantize_row(float4 x, float *scale)
{
    unsigned m = dpp_max16(max4_bits(0u, x));
    if (HD == 128) m = max(m, (unsigned)__shfl_xor((int)m, 16));
    float r;
    quantize_scale(m, &r, scale);
    return finite_bits(m) ? quantize4(x, r) : 0;
}

// Where token row r of a packed batch goes: its sequence (-1: none has it),
// cache row, rotary position, and whether its sequence is skipped.
struct TokenPlace {
    int seq, row, at;
    bool skip;
};
__device__ __forceinline__ TokenPlace find_token(const ManyArgs &a, int r, int lane)
{
    TokenPlace t{-1, 0, 0, false};
    if (!a.begin) {
        t.seq = r;
        t.row = t.at = a.pos ? a.pos[r] : a.pos_scalar;
        t.skip = t.row < 0 || t.row > a.max_pos;
        return t;
    }
    bool stop = false;
    for (int base = 0; base < a.n_seq && !stop && t.seq < 0; base += kWave) {
        const SeqLane s = seq_lane(a, base, lane, &stop);
        const int i = base + lane;
        // (a skipped sequence's rows by its own two bounds)
        const bool has = i < a.n_seq && s.first <= r && r < a.begin[i + 1];
        const uint64_t who = __builtin_amdgcn_ballot_w64(has);
        if (!who) continue;
        const int l = __builtin_ctzll(who);
        t.seq = base + l;
        t.skip = __builtin_amdgcn_readlane(s.n, l) < 0;
        const int j = r - __builtin_amdgcn_readlane(s.first, l);
        t.row = t.at = __builtin_amdgcn_readlane(s.p0, l) + j;
        if (a.parent && !t.skip) {
            const TreeLane w = tree_lane(a.parent + (r - j), __builtin_amdgcn_readlane(s.n, l), lane);
            const int depth = (int)__popcll(w.sees);
            t.at = t.row - j + __builtin_amdgcn_readlane(depth, j) - 1;
        }
    }
    if (t.seq < 0 && stop) t = TokenPlace{0, 0, 0, true};  // behind a begin that goes back
    return t;
}
template <int HD>
__device__ __forceinline__ void fill_nan(float *out, size_t first4, int n4, int i0, int step)
{
    const float nan = __uint_as_float(0x7fc00000u);
    for (int i = i0; i < n4; i += step) reinterpret_cast<float4 *>(out)[first4 + i] = make_float4(nan, nan, nan, nan);
}

// A head row of the cache, LR = HD / 4 lanes of a float4 each: element i of
// the [kv_dim / 4] words of (seq, row).  8 bits: q and sc are what
// quantize_row gives.
template <int HD, bool Q8>
__device__ __forceinline__ void store_row(const ManyArgs &a, int seq, int row, int i, float4 x, int q, float sc, bool value)
{
    constexpr int LR = HD / 4;
    const size_t to = (size_t)seq * a.seq_stride + (size_t)row * (a.n_kv_heads * HD);
    if constexpr (Q8) {
        reinterpret_cast<int *>((value ? a.v8 : a.k8) + to)[i] = q;
        if ((i & (LR - 1)) == 0)
            (value ? a.vs : a.ks)[(size_t)seq * a.scale_stride + (size_t)(i / LR) * a.scale_rows + row] = sc;
    } else {
        reinterpret_cast<float4 *>((value ? a.v_cache : a.k_cache) + to)[i] = x;
    }
}

// A wave per token: its K rows rotated and its V rows as they are, into
// cache row p0 + j of its sequence; NaN into the output rows of skipped
// sequences.  Rows behind the last sequence are left alone.  For calls of
// many tokens a sequence, whose tiles read each other's rows; for few, the
// attention kernel does it (fused), one launch less.  Bound by memory at 8192
// tokens of 8 heads of 128 (26.8 us, 5.2 TB/s), by latency at 400 (5.6 us).
template <int HD, bool Q8>
__global__ __launch_bounds__(kAppendWaves * kWave) void many_append_kernel(ManyArgs a)
{
    const int lane = threadIdx.x & (kWave - 1);
    const int r = blockIdx.x * kAppendWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (r >= a.n_tokens) return;
    constexpr int LR = HD / 4, kAhead = 4;  // lanes of a head row, words a lane has on their way
    const int words = a.n_kv_heads * LR;
    const float4 *kn = reinterpret_cast<const float4 *>(a.k_new) + (size_t)r * words;
    const float4 *vn = reinterpret_cast<const float4 *>(a.v_new) + (size_t)r * words;
    float4 k[kAhead], v[kAhead];
    auto load = [&](int first) {
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            const int i = first + kWave * u + lane;
            k[u] = i < words ? kn[i] : make_float4(0, 0, 0, 0);
            v[u] = i < words ? vn[i] : make_float4(0, 0, 0, 0);
        }
    };
    load(0);  // (ahead of the token's place)
    const TokenPlace t = find_token(a, r, lane);
    if (t.seq < 0) return;
    if (t.skip) {
        fill_nan<HD>(a.out, (size_t)r * a.n_heads * LR, a.n_heads * LR, lane, kWave);
        return;
    }
    const float4 turn = a.rope[(size_t)t.at * LR + (lane & (LR - 1))];
    for (int first = 0; first < words; first += kWave * kAhead) {
        if (first) load(first);
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            const int i = first + kWave * u + lane;
            if (i >= words) break;
            const float4 y = rope4(k[u], turn);
            float sk = 0.0f, sv = 0.0f;
            const int qk = Q8 ? quantize_row<HD>(y, &sk) : 0, qv = Q8 ? quantize_row<HD>(v[u], &sv) : 0;
            store_row<HD, Q8>(a, t.seq, t.row, i, y, qk, sk, false);
            store_row<HD, Q8>(a, t.seq, t.row, i, v[u], qv, sv, true);
        }
    }
}

// ---- the attention kernel -----------------------------------------------------

// The new rows of a chunk in a fused call, K and V by token, as the cache
// holds them (rows 16 bytes apart in their banks).
template <int HD, bool Q8, int N>
struct NewRows {
    float x[2][N][HD + 4];
};
template <int HD, int N>
struct NewRows<HD, true, N> {
    int x[2][N][HD / 4 + 4];
    float scale[2][N];
};

constexpr int kManyRows = 16;   // rows of a tile of many_attention_kernel
constexpr int kWideRows = 256;  // and of wide_attention_kernel
constexpr int kSmallNew = 32;   // new tokens of a sequence that fused calls of the former hold

template <int HD, int W, bool Q8, bool STEP>
struct ManyShared {
    union {
        struct {
            half8v q[HD / 32][2][kWave];     // Q's operand: high and low halves
            NewRows<HD, Q8, STEP ? 1 : kSmallNew> fresh;
        };
        float o[W][kManyRows][HD + 4];       // the waves' outputs
        struct {
            float w[kManyRows][kManySplits + 1];  // the merge: weights of a row's records
            float4 part[W * kWave];               // and partial sums of them
        } merge;
    };
    float qf[kManyRows];                     // 2^(e - 13) log2(e) / sqrt(HD) of each row (NaN: a row without result)
    float m[W][kManyRows], l[W][kManyRows];
    float unit[W][kManyRows];                // O's unit of each wave and row
    float kf[W][kTileKeys];                  // fp32: K's factors of each wave's tile
    uint64_t sees[STEP ? 1 : kTreeMax], bad;  // tree_lane of each node, and the bad ones
    int last;
};

// O's unit in a row is a power of two, and a probability times its value row's
// factor over it goes into fp16 halves, which hold 2^-25 at least and 2^15 with
// room.  Whether a tile leaves it, and the reference of the softmax, as they
// are: mt is the largest score, and the exponent of `most` at least that of any
// factor over the unit (of positions seen or not; NaN or infinite: it does not).
__device__ __forceinline__ bool fits_unit(float mt, float ref, float most)
{
    // mt <= ref + 8, and mt - ref + 7 + (e - 127) <= 15
    const float e = (float)max((int)(__float_as_uint(most) >> 23), 127);
    return __builtin_fmaf(most, 0.0f, mt) + e <= ref + (kProbRoom + 127.0f);
}
// And where it does not, the unit's exponent: top 2^16 is the row's largest
// product in the tile, `up` by how much the reference moved, which takes 2^-up
// off what O holds.  With products of 2^15 units and more it goes up, to where
// they are near 2^6.  With less than 2^5 after the reference moved (so that
// they may be all that the row is made of) it goes down as far; but not by over
// 2^60 more than O loses, which then outweighs them.
__device__ __forceinline__ int next_unit(int unit, float top, float up)
{
    const int e = (int)(__float_as_uint(top) >> 23) - 127 + kRoom - unit;
    if (e < 15 && (up == 0.0f || e >= 5)) return unit;
    return min(max(unit + e - 6, max(kLeastUnit, unit - (int)fminf(up + 60.0f, 300.0f))), 126);
}

// max / sum of a lane's value and those of the lanes 16, 32 and 48 away (the
// swaps of one register with itself would be folded: each takes a copy)
template <bool MAX>
__device__ __forceinline__ float rows4(float x)
{
    auto op = [](float a, float b) { return MAX ? fmaxf(a, b) : a + b; };
    float y = x;
    asm("" : "+v"(y));
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    x = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    y = x;
    asm("" : "+v"(y));
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return op(__uint_as_float(t[0]), __uint_as_float(t[1]));
}

__device__ __forceinline__ unsigned rows4_bits(unsigned x)
{
    unsigned y = x;
    asm("" : "+v"(y));
    const auto r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
    x = max((unsigned)r[0], (unsigned)r[1]);
    y = x;
    asm("" : "+v"(y));
    const auto t = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    return max((unsigned)t[0], (unsigned)t[1]);
}

// The sum of a tile's records, for R rows from R rb on, by T >= 16 R threads:
// record s of row i counts 2^(lse_s - max lse) / their sum.
template <int HD, int BM, int R, int T, typename Merge>
__device__ __forceinline__ void merge_rows(const ManyArgs &a, Merge &sh, int gi, int n_split, const Place &p, int kvh, int rb,
                                           int tid)
{
    constexpr int LR = HD / 4;
    const int rows = p.n * a.group, r0 = p.tile * BM + R * rb;
    if (r0 >= rows) return;
    const size_t rec0 = (size_t)gi * a.splits * BM + R * rb;
    const float ninf = -__builtin_inff();
    // the rows' float4 words, `items` of them; with fewer than threads the
    // records are dealt to `parts` threads a word
    const int items = min(R, rows - r0) * LR;
    int parts = 1;
    while (2 * parts * items <= T) parts *= 2;
    const auto wr = make_rsrc(a.ws_o + rec0 * HD, (uint32_t)n_split * BM * HD * 4u);
    const int part = parts > 1 ? tid / items : 0;
    float4 x[8];
    auto load = [&](int i, int s) {  // (past the last record: 0)
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = buf_load4<kSc1>(wr, (uint32_t)((s + k * parts) * BM * HD + 4 * i) * 4u);
    };
    load(tid - part * items, part);  // on their way while the weights are formed
    if (T == 16 * R || tid < 16 * R) {
        const int row = tid >> 4, l = tid & 15;
        const auto lr = make_rsrc(a.ws_lse + rec0, (uint32_t)n_split * BM * 4u);
        float y[kManySplits / 16], top = ninf;
#pragma unroll
        for (int k = 0; k < kManySplits / 16; k++) {
            const int s = l + 16 * k;
            y[k] = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(lr, (s * BM + row) * 4, 0, kSc1));
            if (s >= n_split) y[k] = ninf;
        }
#pragma unroll
        for (int k = 0; k < kManySplits / 16; k++) top = fmaxf(top, y[k]);
        top = fmaxf(top, dpp<0x121>(top));
        top = fmaxf(top, dpp<0x122>(top));
        top = fmaxf(top, dpp<0x124>(top));
        top = fmaxf(top, dpp<0x128>(top));
        if (top == ninf) top = 0.0f;
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < kManySplits / 16; k++) {
            y[k] = fast_exp2(y[k] - top);
            sum += y[k];
        }
        sum += dpp<0x121>(sum);
        sum += dpp<0x122>(sum);
        sum += dpp<0x124>(sum);
        sum += dpp<0x128>(sum);
        const float inv = 1.0f / sum;
#pragma unroll
        for (int k = 0; k < kManySplits / 16; k++)
            if (l + 16 * k < n_split) sh.w[row][l + 16 * k] = y[k] * inv;
    }
    __syncthreads();
    for (int i0 = 0; i0 < items; i0 += T) {
        const int i = i0 + tid - part * items, row = i / LR;
        const bool mine = i < items && part < parts;
        float4 acc = make_float4(0, 0, 0, 0);
        for (int s = part; s < n_split; s += 8 * parts) {
            if (i0 > 0 || s != part) load(i, s);
            if (mine)
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (s + k * parts < n_split) fma4(acc, sh.w[row][s + k * parts], x[k]);
        }
        if (parts > 1) {
            sh.part[tid] = acc;
            __syncthreads();
            if (part == 0 && mine)
                for (int t = 1; t < parts; t++) fma4(acc, 1.0f, sh.part[t * items + i]);
        }
        if (part == 0 && mine) {
            const int r = r0 + row;
            const int j = (int)fast_div((uint32_t)r, a.by_group);
            const int head = kvh * a.group + r - j * a.group;
            reinterpret_cast<float4 *>(a.out)[((size_t)(p.first + j) * a.n_heads + head) * LR + (i - row * LR)] = acc;
        }
    }
}

// Tiles of 16 rows, W waves.  STEP: calls of one token a sequence (begin
// NULL), whose rows all see the whole chunk.
//
// Short calls are latency: the launch, the rows of q, a pass or two of W x 32
// positions, the records (3 us).  A pass is bound by its vector instructions,
// about 500 a wave at head_dim 128 over 8 bits (900 in fp32) beside 32 (48)
// products, half of them making fp16 operands of what comes from memory; 16
// rows share them.  Eight waves for 8 bits, whose passes are short (one
// workgroup a CU then holds 64 KB of rows on their way), four in fp32.
// Measured under graph replay over several layers, heads/KV heads/head_dim, us:
// 8-bit step 32/4/64 at 256 5.7, 32/8/128 at 4096 11.2 and at 65536 36.5 (3.8
// TB/s), 32 sequences at 4096 63 (4.3 TB/s; one layer again and again 52);
// fp32 tree of 8 at 258 32/4/64 10.6, of 31 at 1024 32/8/128 23.0.
template <int HD, int W, bool Q8, bool STEP>
__global__ __launch_bounds__(W * kWave, HD == 128 && !Q8 ? 1 : 2) void many_attention_kernel(ManyArgs a)
{
    constexpr int BM = kManyRows, KS = HD / 32, VB = HD / 16, LR = HD / 4;
    constexpr int kThreads = W * kWave, kPassKeys = W * kTileKeys;
    __shared__ ManyShared<HD, W, Q8, STEP> sh;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int m = lane & 15, g = lane >> 4;

    // the workgroup's tile, KV head and chunk: a (tile, KV head) group's
    // chunks on one XCD, or (spread) on all
    const int n_groups = a.slots * a.n_kv_heads;
    int gi, split;
    if (a.spread) {
        split = blockIdx.x / n_groups;
        gi = blockIdx.x - split * n_groups;
    } else {
        const int local = blockIdx.x / kXcds;
        const int gl = (int)fast_div((uint32_t)local, a.by_splits);
        split = local - gl * a.splits;
        gi = gl * kXcds + (blockIdx.x & (kXcds - 1));
    }
    if (!STEP && a.fused && blockIdx.x == 0) {
        // skipped sequences' output rows, if there are any
        bool stop = false, any = false;
        for (int base = 0; base < a.n_seq && !stop && !any; base += kWave)
            any = __builtin_amdgcn_ballot_w64(seq_lane(a, base, lane, &stop).n < 0) != 0;
        if (any)
            for (int r = wave; r < a.n_tokens; r += W) {
                const TokenPlace t = find_token(a, r, lane);
                if (t.seq >= 0 && t.skip)
                    fill_nan<HD>(a.out, (size_t)r * a.n_heads * LR, a.n_heads * LR, lane, kWave);
            }
    }
    if (gi >= n_groups) return;
    const int slot = (int)fast_div((uint32_t)gi, a.by_kv_heads);
    const int kvh = gi - slot * a.n_kv_heads;
    Place p;
    if constexpr (STEP) {
        const int p0 = a.pos ? a.pos[slot] : a.pos_scalar;
        if (p0 < 0 || p0 > a.max_pos) {
            if (split == 0)
                fill_nan<HD>(a.out, ((size_t)slot * a.n_heads + kvh * a.group) * LR, a.group * LR, tid, kThreads);
            return;
        }
        p = Place{slot, 0, slot, 1, p0};
    } else {
        p = find_place<BM>(a, slot, lane);
        if (p.seq < 0) return;
    }
    const int rows = p.n * a.group, r0 = p.tile * BM, n_rows = min(BM, rows - r0);
    const int j0 = STEP ? 0 : (int)fast_div((uint32_t)r0, a.by_group);
    const int j1 = STEP ? 0 : min(p.n - 1, (int)fast_div((uint32_t)(r0 + BM - 1), a.by_group));
    const bool tree = !STEP && a.parent, fused = STEP || a.fused;
    const int kv_end = tree ? p.p0 + p.n : p.p0 + j1 + 1;
    const int c0 = split * a.chunk, c1 = min(kv_end, c0 + a.chunk);
    if (c0 >= kv_end) return;

    // ---- the cache's rows ----
    const int kv_dim = a.n_kv_heads * HD;
    const uint32_t row_bytes = (uint32_t)kv_dim * (Q8 ? 1 : 4), head_off = (uint32_t)kvh * HD * (Q8 ? 1 : 4);
    const size_t base = (size_t)p.seq * a.seq_stride;
    const int old1 = fused ? min(c1, p.p0) : c1;           // cached rows of the chunk: up to here
    const uint32_t bytes = (uint32_t)old1 * row_bytes;     // (rows from there on read as zero)
    const auto kr = Q8 ? make_rsrc(a.k8 + base, bytes) : make_rsrc(a.k_cache + base, bytes);
    const auto vr = Q8 ? make_rsrc(a.v8 + base, bytes) : make_rsrc(a.v_cache + base, bytes);
    const size_t sbase = (size_t)p.seq * a.scale_stride + (size_t)kvh * a.scale_rows;
    const auto ksr = make_rsrc(Q8 ? a.ks + sbase : nullptr, Q8 ? (uint32_t)old1 * 4u : 0u);
    const auto vsr = make_rsrc(Q8 ? a.vs + sbase : nullptr, Q8 ? (uint32_t)old1 * 4u : 0u);

    constexpr int KR = Q8 ? HD / 64 : HD / 16, VR = Q8 ? 1 : HD / 64;
    float4 kraw[2][KR], vraw[8][VR];
    float2 vraw8[8];
    float4 ksc[2], vsc[2];
    const uint32_t k_lane = m * row_bytes + head_off + 16 * g;
    const uint32_t v_lane = 4 * g * row_bytes + head_off + (Q8 ? HD / 16 : 16) * m;
    auto load_k = [&](int key0) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const uint32_t off = k_lane + (uint32_t)(key0 + 16 * b) * row_bytes;
#pragma unroll
            for (int i = 0; i < KR; i++) kraw[b][i] = buf_load4(kr, off + 64 * i);
            if constexpr (Q8) ksc[b] = buf_load4(ksr, (uint32_t)(key0 + 16 * b + 4 * g) * 4u);
        }
    };
    auto load_v = [&](int key0) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t off = v_lane + (uint32_t)(key0 + 16 * (j >> 2) + (j & 3)) * row_bytes;
            if constexpr (Q8) {
                if constexpr (HD == 128)
                    vraw8[j] = buf_load2(vr, off);
                else
                    vraw8[j].x = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(vr, (int)off, 0, 0));
            } else {
#pragma unroll
                for (int i = 0; i < VR; i++) vraw[j][i] = buf_load4(vr, off + 256 * i);
            }
        }
        if constexpr (Q8)
#pragma unroll
            for (int b = 0; b < 2; b++) vsc[b] = buf_load4(vsr, (uint32_t)(key0 + 16 * b + 4 * g) * 4u);
    };
    // The chunk's new rows: tokens [t0, t0 + n_new).
    const int t0 = fused ? max(c0 - p.p0, 0) : 0, n_new = fused ? max(min(c1 - p.p0, p.n) - t0, 0) : 0;
    auto is_new = [&](int j) { return (unsigned)(j - t0) < (unsigned)n_new; };
    // The rows of a tile that this call brings, in place of what was read.
    auto fresh_k = [&](int key0) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int j = key0 + 16 * b + m - p.p0;
            if (is_new(j)) {
#pragma unroll
                for (int i = 0; i < KR; i++)
                    kraw[b][i] = *reinterpret_cast<const float4 *>(&sh.fresh.x[0][STEP ? 0 : j][16 * i + 4 * g]);
            }
            if constexpr (Q8)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int t = key0 + 16 * b + 4 * g + i - p.p0;
                    if (is_new(t)) {
                        (&ksc[b].x)[i] = sh.fresh.scale[0][STEP ? 0 : t];
                        (&vsc[b].x)[i] = sh.fresh.scale[1][STEP ? 0 : t];
                    }
                }
        }
    };
    auto fresh_v = [&](int key0) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int t = key0 + 16 * (j >> 2) + 4 * g + (j & 3) - p.p0;
            if (is_new(t)) {
                const int at = STEP ? 0 : t;
                if constexpr (Q8) {
                    if constexpr (HD == 128)
                        vraw8[j] = *reinterpret_cast<const float2 *>(&sh.fresh.x[1][at][2 * m]);
                    else
                        vraw8[j].x = __int_as_float(sh.fresh.x[1][at][m]);
                } else {
#pragma unroll
                    for (int i = 0; i < VR; i++)
                        vraw[j][i] = *reinterpret_cast<const float4 *>(&sh.fresh.x[1][at][64 * i + 4 * m]);
                }
            }
        }
    };

    // ---- the tile's rows of Q and the chunk's new rows ----
    // LR threads a row: rows of Q first, then new K rows, then new V rows.
    // The loads go out in the order they are needed: these rows', then the
    // first tile's.
    const int lr = tid & (LR - 1), n_jobs = n_rows + 2 * n_new;
    auto token_of = [&](int job) {
        return job < n_rows ? (STEP ? 0 : (int)fast_div((uint32_t)(r0 + job), a.by_group))
                            : t0 + (job - n_rows < n_new ? job - n_rows : job - n_rows - n_new);
    };
    auto load_row = [&](int job) {
        const int j = token_of(job);
        const float *src = job < n_rows ? a.q + ((size_t)(p.first + j) * a.n_heads + kvh * a.group + r0 + job - j * a.group) * HD
                                        : (job < n_rows + n_new ? a.k_new : a.v_new) + ((size_t)(p.first + j) * a.n_kv_heads + kvh) * HD;
        return reinterpret_cast<const float4 *>(src)[lr];
    };
    auto load_turn = [&](int job, int at) {
        return job < n_rows + n_new ? a.rope[(size_t)at * LR + lr] : make_float4(1, 0, 1, 0);
    };
    int key0 = c0 + wave * kTileKeys;
    constexpr int kJobs = kThreads / LR;
    auto pos_of = [&](int job) {
        const int j = token_of(job);
        return p.p0 + (tree ? (int)__popcll(sh.sees[j]) - 1 : j);
    };
    float4 y = make_float4(0, 0, 0, 0), turn = y;
    int job = tid / LR;
    if (job < n_jobs) {
        y = load_row(job);
        if (!tree) turn = load_turn(job, pos_of(job));
    }
    if (key0 < c1) {
        load_k(key0);
        load_v(key0);
    }
    if (tree) {
        if (wave == W - 1) {
            const TreeLane t = tree_lane(a.parent + p.first, p.n, lane);
            sh.sees[lane] = t.sees;
            const uint64_t bad = __builtin_amdgcn_ballot_w64(t.bad);
            if (lane == 0) sh.bad = bad;
        }
        __syncthreads();
    }
    const bool stores = r0 + BM >= rows;  // the last tile sees all new rows: it puts them into the cache
    if (tree && job < n_jobs) turn = load_turn(job, pos_of(job));
    for (; job < n_jobs; job += kJobs) {
        float4 y1 = make_float4(0, 0, 0, 0), turn1 = y1;  // the next one's, on their way
        if (job + kJobs < n_jobs) {
            y1 = load_row(job + kJobs);
            turn1 = load_turn(job + kJobs, pos_of(job + kJobs));
        }
        if (job < n_rows) {
            // rotated, split, and where the products' B operand has it: the
            // contraction takes the dims in an order such that a K load
            // instruction reads whole 64-byte pieces of its rows
            const float4 x = rope4(y, turn);
            unsigned mx = dpp_max16(max4_bits(0u, x));
            if constexpr (HD == 128) mx = max(mx, (unsigned)__shfl_xor((int)mx, 16));
            const bool good = finite_bits(mx) && !(tree && (sh.bad >> token_of(job) & 1));
            const int e = tile_exp(good ? mx : 0u);
            const float sc = good ? exp2_int(13 - e) : 0.0f;
            half2v h[2], l[2];
            split2(x.x * sc, x.y * sc, h[0], l[0]);
            split2(x.z * sc, x.w * sc, h[1], l[1]);
            const int d = 4 * lr;
            const int s = Q8 ? 2 * (d >> 6) + ((d >> 3) & 1) : d >> 5, gg = Q8 ? (d >> 4) & 3 : (d >> 2) & 3;
            const int half = Q8 ? (d >> 2) & 1 : (d >> 4) & 1;
            u32x2 *to = reinterpret_cast<u32x2 *>(&sh.q[s][0][16 * gg + job]) + half;
            to[0] = u32x2{__builtin_bit_cast(unsigned, h[0]), __builtin_bit_cast(unsigned, h[1])};
            to[2 * kWave] = u32x2{__builtin_bit_cast(unsigned, l[0]), __builtin_bit_cast(unsigned, l[1])};
            if (lr == 0) sh.qf[job] = good ? exp2_int(e - 13) * a.scale_log2 : __uint_as_float(0x7fc00000u);
        } else {
            const int j = token_of(job);
            const bool value = job >= n_rows + n_new;
            if (!value) y = rope4(y, turn);
            int q = 0;
            float sc = 0.0f;
            if constexpr (Q8) {
                q = quantize_row<HD>(y, &sc);
                sh.fresh.x[value][STEP ? 0 : j][lr] = q;
                if (lr == 0) sh.fresh.scale[value][STEP ? 0 : j] = sc;
            } else {
                *reinterpret_cast<float4 *>(&sh.fresh.x[value][j][4 * lr]) = y;
            }
            if (stores) store_row<HD, Q8>(a, p.seq, p.p0 + j, kvh * LR + lr, y, q, sc, value);
        }
        y = y1;
        turn = turn1;
    }
    __syncthreads();
    half8v qh[KS], ql[KS];
#pragma unroll
    for (int s = 0; s < KS; s++) {
        qh[s] = sh.q[s][0][lane];
        ql[s] = sh.q[s][1][lane];
    }
    const float qf = sh.qf[m];

    f32x4 o[VB];
    float mrun = kNothing, lrun = 0.0f;
#pragma unroll
    for (int v = 0; v < VB; v++) o[v] = f32x4{0, 0, 0, 0};
    int erun = 0;  // O's unit in the lane's row is 2^(erun - 12) (8 bits: 2^erun, and values are 2^-9 times theirs)

    for (; key0 < c1; key0 += kPassKeys) {
        // ---- scores ----
        const bool fresh = n_new > 0 && key0 + kTileKeys > p.p0;
        if (fresh) fresh_k(key0);
        unsigned badkeys = 0;  // positions of the tile whose key or value is not finite (bit: position - key0)
        float kscale[2];
        if constexpr (!Q8) {
            // each position by its own largest element (block b: position 16 b + m)
            unsigned top[2];
#pragma unroll
            for (int b = 0; b < 2; b++) {
                float x = 0.0f;
#pragma unroll
                for (int i = 0; i < KR; i++) x = max4_abs(x, kraw[b][i]);
                top[b] = rows4_bits(__float_as_uint(x));
            }
            if (__builtin_expect(__builtin_amdgcn_ballot_w64(!finite_bits(max(top[0], top[1]))) != 0, 0)) {
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    unsigned mk = 0;
                    bool bad = false;
#pragma unroll
                    for (int i = 0; i < KR; i++) {
                        bad |= zero_bad(kraw[b][i]);
                        mk = max4_bits(mk, kraw[b][i]);
                    }
                    uint64_t w = __builtin_amdgcn_ballot_w64(bad);
                    w |= w >> 32;
                    w |= w >> 16;
                    badkeys |= (unsigned)(w & 0xffffu) << (16 * b);
                    top[b] = rows4_bits(mk);
                }
            }
#pragma unroll
            for (int b = 0; b < 2; b++) {
                const int e = tile_exp(top[b]);
                kscale[b] = exp2_int(13 - e);
                sh.kf[wave][16 * b + m] = exp2_int(e - 13);
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        }
        f32x4 sc[2], sl[2];  // (two accumulators each: products that add to the one before them wait for it)
#pragma unroll
        for (int b = 0; b < 2; b++) sc[b] = sl[b] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int b = 0; b < 2; b++) {
                half8v kh, kl;
                if constexpr (Q8) {
                    const float4 w = kraw[b][s >> 1];
                    kh = (s & 1) ? bytes_half8(__float_as_uint(w.z), __float_as_uint(w.w))
                                 : bytes_half8(__float_as_uint(w.x), __float_as_uint(w.y));
                } else {
                    const float4 f = make_float4(kscale[b], kscale[b], kscale[b], kscale[b]);
                    split8(mul4(kraw[b][2 * s], f), mul4(kraw[b][2 * s + 1], f), kh, kl);
                }
                sl[b] = mfma16(kh, ql[s], sl[b]);
                sc[b] = mfma16(kh, qh[s], sc[b]);
                if constexpr (!Q8) sl[b] = mfma16(kl, qh[s], sl[b]);
            }
        // K's and V's factors of the lane's positions 16 b + 4 g + i
        float4 kscv[2], vscv[2];
        if constexpr (Q8) {
#pragma unroll
            for (int b = 0; b < 2; b++) {
                // a row's two scales: NaN in either marks it (and V's is then
                // 0 here, which a masked probability may meet)
                auto f = [](float x) { return fmaxf(x, 0.0f) * exp2_int(-kRoom); };
                vscv[b] = make_float4(f(vsc[b].x), f(vsc[b].y), f(vsc[b].z), f(vsc[b].w));
                kscv[b] = make_float4(ksc[b].x + 0.0f * vsc[b].x, ksc[b].y + 0.0f * vsc[b].y,
                                      ksc[b].z + 0.0f * vsc[b].z, ksc[b].w + 0.0f * vsc[b].w);
            }
        } else {
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
            for (int b = 0; b < 2; b++) kscv[b] = *reinterpret_cast<const float4 *>(&sh.kf[wave][16 * b + 4 * g]);
        }
        load_k(key0 + kPassKeys);
        if (fresh) fresh_v(key0);
        float4 vin[2];  // fp32: what V's rows are multiplied by
        if constexpr (!Q8) {
            unsigned top[8], all = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float x = 0.0f;
#pragma unroll
                for (int i = 0; i < VR; i++) x = max4_abs(x, vraw[j][i]);
                top[j] = dpp_max16(__float_as_uint(x));
                all = max(all, top[j]);
            }
            if (__builtin_expect(__builtin_amdgcn_ballot_w64(!finite_bits(all)) != 0, 0)) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    unsigned mv = 0;
                    bool bad = false;
#pragma unroll
                    for (int i = 0; i < VR; i++) {
                        bad |= zero_bad(vraw[j][i]);
                        mv = max4_bits(mv, vraw[j][i]);
                    }
                    top[j] = dpp_max16(mv);
                    const uint64_t w = __builtin_amdgcn_ballot_w64(bad);
                    for (int gg = 0; gg < 4; gg++)
                        if ((w >> (16 * gg)) & 0xffffu) badkeys |= 1u << (16 * (j >> 2) + 4 * gg + (j & 3));
                }
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int e = tile_exp(top[j]);
                (&vscv[j >> 2].x)[j & 3] = exp2_int(e - 1 - kRoom);
                (&vin[j >> 2].x)[j & 3] = exp2_int(13 - e);
            }
        }

        // ---- softmax ----
        float s[8];
#pragma unroll
        for (int t = 0; t < 8; t++) {
            const int b = t >> 2, i = t & 3;
            s[t] = (sc[b][i] + sl[b][i]) * ((&kscv[b].x)[i] * qf);
        }
        if (__builtin_expect(badkeys != 0, 0))
#pragma unroll
            for (int t = 0; t < 8; t++)
                if ((badkeys >> (16 * (t >> 2) + 4 * g + (t & 3))) & 1) s[t] = __uint_as_float(0x7fc00000u);
        if (key0 + kTileKeys > c1 || (!STEP && key0 + kTileKeys - 1 > (tree ? p.p0 - 1 : p.p0 + j0))) {
            // visible: up to `limit`, and of a tree's nodes those of `sees`
            int limit = c1 - 1;
            uint64_t sees = 0;
            if constexpr (!STEP) {
                const int tok = (int)fast_div((uint32_t)min(r0 + m, rows - 1), a.by_group);
                limit = p.p0 + tok;
                if (tree) {
                    limit = p.p0 - 1;
                    sees = sh.sees[tok];
                }
            }
#pragma unroll
            for (int t = 0; t < 8; t++) {
                const int key = key0 + 16 * (t >> 2) + 4 * g + (t & 3);
                const bool see = key <= limit || (!STEP && ((sees >> ((key - p.p0) & 63)) & 1));
                if (!see || key >= c1) s[t] = -__builtin_inff();
            }
        }
        // The reference, a whole number, moves only when a score exceeds it by
        // more than 2^8, and O's unit where a product passes 2^15 of it: most
        // tiles leave both, O and the sum as they are, and need no maximum over
        // the row's lanes.
        auto largest = [&]() {
            return fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
        };
        float mt = largest(), up = 0.0f;
        const bool moves = __builtin_amdgcn_ballot_w64(mt > mrun + kProbRoom) != 0;
        if (moves) {
            mt = rows4<true>(mt);
            const float now = mt > mrun + kProbRoom ? ceilf(mt) : mrun;
            up = now - mrun;
            lrun *= fast_exp2(-up);
            mrun = now;
        }
        const float off = mrun - kProbBias;
        // Probabilities times their value rows' factors (2^-16 of them: these
        // products are finite, and as small as fp32 holds).
#pragma unroll
        for (int t = 0; t < 8; t++) {
            const float x = fast_exp2(s[t] - off);
            lrun += x;
            s[t] = x * (&vscv[t >> 2].x)[t & 3];
        }
        float top = largest();
        if (moves || __builtin_amdgcn_ballot_w64(top > exp2_int(erun - kRoom + 15))) {
            const int now = next_unit(erun, rows4<true>(top), up);
            const float os = fast_exp2((float)(erun - now) - up);
            erun = now;
#pragma unroll
            for (int v = 0; v < VB; v++) o[v] *= os;
        }
        const float vscale = exp2_int(kRoom - erun);
#pragma unroll
        for (int t = 0; t < 8; t++) s[t] *= vscale;
        Half8 h, l;
#pragma unroll
        for (int t = 0; t < 8; t += 2) split2(s[t], s[t + 1], h.h[t / 2], l.h[t / 2]);
        const half8v ph = h.v, pl = l.v;

        // ---- weighted values ----
#pragma unroll
        for (int v = 0; v < VB; v++) {
            half8v vh, vl;
            if constexpr (Q8) {
                Half8 r;
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const unsigned x = __float_as_uint(v < 4 ? vraw8[j].x : vraw8[j].y) ^ 0x80808080u;
                    const unsigned z = __float_as_uint(v < 4 ? vraw8[j + 1].x : vraw8[j + 1].y) ^ 0x80808080u;
                    const unsigned sel = 0x0c000c00u | (unsigned)(4 + (v & 3)) << 16 | (unsigned)(v & 3);
                    r.h[j / 2] = bytes_small(__builtin_amdgcn_perm(z, x, sel));
                }
                vh = r.v;
            } else {
                const int i = v >> 2, c = v & 3;
                auto at = [&](int j) { return (&vraw[j][i].x)[c]; };
                split8(mul4(make_float4(at(0), at(1), at(2), at(3)), vin[0]),
                       mul4(make_float4(at(4), at(5), at(6), at(7)), vin[1]), vh, vl);
            }
            o[v] = mfma16(vh, pl, o[v]);
            if constexpr (!Q8) o[v] = mfma16(vl, ph, o[v]);
            o[v] = mfma16(vh, ph, o[v]);
        }
        load_v(key0 + kPassKeys);
    }

    // ---- the waves' results together ----
    lrun = rows4<false>(lrun);
    __syncthreads();  // (Q's operand is read; its memory takes the outputs)
    if (g == 0) {
        sh.m[wave][m] = mrun;
        sh.l[wave][m] = lrun;
        sh.unit[wave][m] = exp2_int(Q8 ? erun : erun - 12);
    }
    // register i of block v: dim (8 bits) VB (4 g + i) + v, or 64 (v / 4) + 4 (4 g + i) + v % 4
#pragma unroll
    for (int v = 0; v < VB; v += 4)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int d = Q8 ? VB * (4 * g + i) + v : 16 * v + 4 * (4 * g + i);
            *reinterpret_cast<float4 *>(&sh.o[wave][m][d]) = make_float4(o[v][i], o[v + 1][i], o[v + 2][i], o[v + 3][i]);
        }
    __syncthreads();
    // (a probability's unit is in both sums)
    const int n_split = a.splits > 1 ? (kv_end + a.chunk - 1) / a.chunk : 1;
    const size_t rec = ((size_t)gi * a.splits + split) * BM;
    for (int i = tid; i < n_rows * LR; i += kThreads) {
        const int row = i / LR, d = (i - row * LR) * 4, r = r0 + row;
        float top = sh.m[0][row];
#pragma unroll
        for (int w = 1; w < W; w++) top = fmaxf(top, sh.m[w][row]);
        float f[W], total = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) {
            f[w] = fast_exp2(sh.m[w][row] - top);
            total += f[w] * sh.l[w][row];
        }
        // (weights before units: their product with a sum of values is no
        // larger than the values, which may fill fp32's range)
        const bool none = total == 0.0f;  // a chunk none of whose positions the row sees: nothing, weight 0
        const float inv = none ? 0.0f : (Q8 ? 0x1p9f : 1.0f) / total;
        float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < W; w++) {
            float4 x = *reinterpret_cast<const float4 *>(&sh.o[w][row][d]);
            scale4(x, f[w] * inv);
            fma4(acc, sh.unit[w][row], x);
        }
        if (n_split == 1) {
            const int j = STEP ? 0 : (int)fast_div((uint32_t)r, a.by_group);
            const int head = kvh * a.group + r - j * a.group;
            *reinterpret_cast<float4 *>(a.out + ((size_t)(p.first + j) * a.n_heads + head) * HD + d) = acc;
        } else {
            *reinterpret_cast<float4 *>(a.ws_o + (rec + row) * HD + d) = acc;
            if (d == 0) a.ws_lse[rec + row] = none ? -__builtin_inff() : top + log2f(total) - kProbBias;
        }
    }
    if (n_split == 1 || a.spread) return;

    // ---- the last chunk to arrive adds up the records ----
    // (all in one XCD's L2: the stores have drained to it, the counter is an
    // L2 atomic, and the loads miss in L1)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
        const int before = __hip_atomic_fetch_add(a.counters + gi, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sh.last = before == n_split - 1;
        if (before == n_split - 1) __hip_atomic_store(a.counters + gi, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (sh.last) merge_rows<HD, BM, BM, kThreads>(a, sh.merge, gi, n_split, p, kvh, 0, tid);
}

// The records of a spread launch's tiles of BM rows added up, R rows a
// workgroup: 4, or 16 where those are four workgroups a CU and more (256-row
// tiles at head_dim 128, us with 4 : 16: 8 trees of 64 nodes of 64/8 heads in
// two chunks 21.2 : 11.8, a tree of 31 nodes of 32/8 heads in 32 chunks
// 7.0 : 9.5).
constexpr int kMergeRows[2] = {4, 16};
template <int HD, int BM, int R>
__global__ __launch_bounds__(256) void many_merge_kernel(ManyArgs a)
{
    __shared__ struct {
        float w[R][kManySplits + 1];
        float4 part[256];
    } sh;
    const int tid = threadIdx.x;
    const int gi = blockIdx.x / (BM / R), rb = blockIdx.x % (BM / R);
    const int slot = (int)fast_div((uint32_t)gi, a.by_kv_heads);
    const int kvh = gi - slot * a.n_kv_heads;
    const Place p = find_place<BM>(a, slot, tid & (kWave - 1));
    if (p.seq < 0 || p.n < 0) return;
    const int j1 = min(p.n - 1, (int)fast_div((uint32_t)(p.tile * BM + BM - 1), a.by_group));
    const int kv_end = a.parent ? p.p0 + p.n : p.p0 + j1 + 1;
    const int n_split = (kv_end + a.chunk - 1) / a.chunk;
    if (n_split > 1) merge_rows<HD, BM, R, 256>(a, sh, gi, n_split, p, kvh, rb, tid);
}

// ---- rows of a cache, moved ---------------------------------------------------

// The accepted paths' rows, moved together (tree_keep): path[i] of sequence
// seq goes from row pos + path[i] to pos + i, in every held layer.  A thread
// has one 16-byte column of one layer's K or V (or, for 8 bits, one head's
// scales) and moves its rows in order: path ascends, so a row is read
// before anything is written over it.
// Bound by latency: 4.7 us for a path of one tree over 16 layers of 8 heads
// of 128, 8 rows on their way at a time.
struct KeepArgs {
    char *k, *v;                       // sequence 0's first layer
    float *ks, *vs;                    // 8 bits: its scales
    const int *pos, *path;
    long long seq_bytes, layer_bytes;  // between sequences, and layers
    long long scale_seq, scale_layer;  // floats
    int row_bytes, scale_rows, n_kv_heads;
    int n_layers, max_path, seq_len;
    int columns;                       // 16-byte columns of a row
};
constexpr int kKeepThreads = 256;
template <typename T>
__device__ __forceinline__ void keep_column(T *col, size_t stride, const int *path, int n)
{
    for (int i = 0; i < n; i += 8) {
        T x[8];
#pragma unroll
        for (int t = 0; t < 8; t++)
            x[t] = col[(size_t)path[min(i + t, n - 1)] * stride];
#pragma unroll
        for (int t = 0; t < 8; t++)
            if (i + t < n) col[(size_t)(i + t) * stride] = x[t];
    }
}
template <bool Q8>
__global__ __launch_bounds__(kKeepThreads) void tree_keep_kernel(KeepArgs a)
{
    __shared__ int path[kTreeMax];
    const int seq = blockIdx.y, tid = threadIdx.x;
    const int p0 = a.pos[seq];
    // (a path ends at its first entry that is not above the one before it, or leaves the cache)
    int n = 0;
    if (tid < kWave) {
        const int x = tid < a.max_path ? a.path[(size_t)seq * a.max_path + tid] : -1;
        const int prev = __shfl_up(x, 1);
        const bool ok = x < kTreeMax && x > (tid ? prev : -1) && p0 >= 0 && p0 < a.seq_len - x;
        const uint64_t bad = __builtin_amdgcn_ballot_w64(!ok);
        n = bad ? __builtin_ctzll(bad) : kWave;
        path[tid] = tid < n ? x : -1;
    }
    __syncthreads();
    if (tid >= kWave) {
        while (n < kTreeMax && path[n] >= 0) n++;
    }
    const int per_layer = 2 * a.columns + (Q8 ? 2 * a.n_kv_heads : 0);
    const int at = blockIdx.x * kKeepThreads + tid;
    if (at >= per_layer * a.n_layers) return;
    const int layer = at / per_layer;
    int c = at - layer * per_layer;
    if (c < 2 * a.columns) {
        char *base = (c < a.columns ? a.k : a.v) + seq * a.seq_bytes + layer * a.layer_bytes + (size_t)p0 * a.row_bytes;
        if (c >= a.columns) c -= a.columns;
        keep_column(reinterpret_cast<f32x4 *>(base + 16 * (size_t)c), (size_t)a.row_bytes / 16, path, n);
    } else {
        c -= 2 * a.columns;
        float *base = (c < a.n_kv_heads ? a.ks : a.vs) + seq * a.scale_seq + layer * a.scale_layer + p0;
        if (c >= a.n_kv_heads) c -= a.n_kv_heads;
        keep_column(base + (size_t)c * a.scale_rows, (size_t)1, path, n);
    }
}

// Rows [row0, row0 + n) of one sequence and layer between fp32 memory and the
// cache: quantised on the way in, what they stand for on the way out.
// Bound by memory: 8192 rows of 8 heads of 128, K and V, in 22 us (3.8 TB/s)
// and out in 15 us (5.7 TB/s); four words a thread on their way instead of
// one took as long.
struct RowsArgs {
    const float *k_in, *v_in;  // (write: either may be NULL)
    float *k_out, *v_out;      // (read)
    int8_t *k8, *v8;           // at row0
    float *ks, *vs;            // at row0 of KV head 0
    int scale_rows, n_kv_heads, n;
};
template <int HD>
__global__ __launch_bounds__(256) void q8_write_kernel(RowsArgs a)
{
    constexpr int LR = HD / 4;
    const int per_row = a.n_kv_heads * LR;
    const long long total = (long long)a.n * per_row;
    const float *in = blockIdx.y ? a.v_in : a.k_in;
    int8_t *to = blockIdx.y ? a.v8 : a.k8;
    float *scales = blockIdx.y ? a.vs : a.ks;
    if (!in) return;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        float s;
        const int q = quantize_row<HD>(reinterpret_cast<const float4 *>(in)[i], &s);
        reinterpret_cast<int *>(to)[i] = q;
        if (((int)i & (LR - 1)) == 0) {
            const int row = (int)(i / per_row), h = (int)(i - (long long)row * per_row) / LR;
            scales[(size_t)h * a.scale_rows + row] = s;
        }
    }
}
template <int HD>
__global__ __launch_bounds__(256) void q8_read_kernel(RowsArgs a)
{
    constexpr int LR = HD / 4;
    const int per_row = a.n_kv_heads * LR;
    const long long total = (long long)a.n * per_row;
    float *out = blockIdx.y ? a.v_out : a.k_out;
    const int8_t *from = blockIdx.y ? a.v8 : a.k8;
    const float *scales = blockIdx.y ? a.vs : a.ks;
    if (!out) return;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const int q = reinterpret_cast<const int *>(from)[i];
        const int row = (int)(i / per_row), h = (int)(i - (long long)row * per_row) / LR;
        const float s = scales[(size_t)h * a.scale_rows + row];
        reinterpret_cast<float4 *>(out)[i] = make_float4((float)(int8_t)q * s, (float)(int8_t)(q >> 8) * s,
                                                         (float)(int8_t)(q >> 16) * s, (float)(q >> 24) * s);
    }
}

}  // namespace leap
