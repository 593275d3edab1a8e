// The selection of a beam search: of all continuations (beam, token) of a
// group of beams, the best by score[beam] + log_softmax(logits[beam])[token].
//
// Two launches.  beam_rows_kernel reads the logits once: a wave takes up to
// 4096 of a row, all loads in flight at once, keeps them in registers, and
// leaves the row's maximum and sum of exponentials over them and their `beams`
// best, in order.  The k-th largest of the lanes' maxima bounds the k-th
// largest of all from below, so that little more than k values are looked at
// one by one.  beam_best_kernel joins a group's records: a wave a row, then all
// rows' best against each other, in 64 bits.
//
// Bound by the logits' bytes (192 rows of 128256: 98.5 MB in 19.7 us, 5.0 TB/s,
// 8 us of it also spent on instructions, 13 a value), or for few rows by two
// launches' latency (4 rows of 32000: 4.1 and 4.7 us).
//
// A row's log sum of exponentials is fp32's over a wave's logits (arguments of
// exp2 rounded, a chain of up to 64 terms a lane), 64 bits' over its waves: up
// to 6e-6 off.
//
// Order: a larger total first; of one beam's equal totals the larger logit,
// then the lower token; of several beams' the lower beam.
#pragma once

#include "paged_attention.hpp"

namespace leap {

constexpr int kBeamMax = 16;                       // beams of a group
constexpr int kBeamUnits = 64;                     // records of a row, at most
constexpr int kBeamWords = 16;                     // float4 words of a row that a lane holds, at most
constexpr int kBeamVocab = kBeamUnits * kBeamWords * 4 * kWave;  // 262144

struct BeamArgs {
    const float *logits, *scores;
    long long stride;               // floats between rows
    int vocab, beams, rows, units;  // records of a row
    uint64_t *keys;                 // [row][unit][beams]
    float2 *sums;                   // [row][unit]: maximum, sum of exponentials over it (NaN: not a distribution)
    int *parent, *token;
    float *best;
};

// A key that orders values descending and, among equal ones, places ascending.
__device__ __forceinline__ uint64_t beam_key(float x, int place)
{
    unsigned b = __float_as_uint(x + 0.0f);  // (-0 as 0)
    b = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (uint64_t)b << 32 | (unsigned)~place;
}
__device__ __forceinline__ float beam_value(uint64_t key)
{
    const unsigned b = (unsigned)(key >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int beam_place(uint64_t key) { return (int)~(unsigned)key; }

// The k-th largest of the lanes' values (as ordered bits).
__device__ __forceinline__ unsigned kth_largest(unsigned mine, int k)
{
    unsigned top = 0;
    for (int i = 0; i < k;) {
        top = wave_max_u32(mine);
        const uint64_t at = __builtin_amdgcn_ballot_w64(mine == top);
        i += (int)__popcll(at);
        if (mine == top) mine = 0;
        if (top == 0) break;
    }
    return top;
}

// U words of four logits a lane.
template <int U>
__global__ __launch_bounds__(256, U == 16 ? 5 : 8) void beam_rows_kernel(BeamArgs a)
{
    // (values and places apart: 6 bytes)
    constexpr int kList = (kBeamMax - 1) * 4 * U;  // values above the bound: in at most k - 1 lanes
    union BeamList {
        uint64_t keys[kWave];
        struct {
            float value[kList];
            uint16_t place[kList], tie[kBeamMax];
        } apart;
    };
    __shared__ BeamList lists[4];
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const long long at = (long long)blockIdx.x * 4 + wave;
    const int row = (int)(at / a.units), unit = (int)(at - (long long)row * a.units);
    if (row >= a.rows) return;
    const float *x_at = a.logits + row * a.stride;
    const int first = unit * (U * 4 * kWave);
    const float ninf = -__builtin_inff();
    float x[U][4];
    // (loads without branches between them: all in flight at once)
    if (first + U * 4 * kWave <= a.vocab) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            f32x4 y;
            __builtin_memcpy(&y, x_at + first + (u * kWave + lane) * 4, 16);  // (rows need not be aligned)
#pragma unroll
            for (int e = 0; e < 4; e++) x[u][e] = y[e];
        }
    } else {
        const int left = a.vocab - first;
        const auto r = make_rsrc(x_at + first, (uint32_t)left * 4u);
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = (u * kWave + lane) * 4 + e;
                const float y = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, i * 4, 0, 0));
                x[u][e] = i < left ? y : ninf;
            }
    }
    float top = ninf;
#pragma unroll
    for (int u = 0; u < U; u++) top = fmaxf(fmaxf(top, fmaxf(x[u][0], x[u][1])), fmaxf(x[u][2], x[u][3]));
    const unsigned mine = (unsigned)(beam_key(top, 0) >> 32);
    const float all = lanes_max(top);
    // a NaN or +inf makes the sum NaN; the maxima pass over a NaN
    float sum = 0.0f;
    if (all > ninf) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) sum += fast_exp2((x[u][e] - all) * 1.44269504088896341f);
    } else {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) sum += x[u][e] != x[u][e] ? x[u][e] : 0.0f;
    }
    sum = lanes_sum(sum);
    const bool odd = sum != sum;
    if (lane == 0) a.sums[at] = make_float2(odd ? sum : all, sum);
    uint64_t *to = a.keys + at * a.beams;
    if (odd) return;  // (its row has no distribution: beam_best_kernel does not look at these)
    const unsigned b = kth_largest(mine, a.beams);
    const float bound = beam_value((uint64_t)b << 32);
    constexpr int H = (4 * U + 31) / 32;
    unsigned hits[H];  // the lane's values from the bound on
    int n = 0;
#pragma unroll
    for (int h = 0; h < H; h++) {
        hits[h] = 0;
#pragma unroll
        for (int j = min(31, 4 * U - 1); j >= 0; j--) hits[h] = hits[h] + hits[h] + (x[8 * h + j / 4][j % 4] >= bound);
        n += __popc(hits[h]);
    }
    const int upto = wave_scan_add(n), all_hits = __builtin_amdgcn_readlane(upto, kWave - 1);
    BeamList &list = lists[wave];
    if (all_hits <= kWave) {
        // as a rule: little more than k.  One a lane, and each one's rank is its place in the record
        int at = upto - n;
#pragma unroll
        for (int h = 0; h < H; h++)
            while (hits[h]) {
                const int j = 32 * h + __builtin_ctz(hits[h]), i = first + (j / 4 * kWave + lane) * 4 + j % 4;
                hits[h] &= hits[h] - 1;
                list.keys[at++] = beam_key(i < a.vocab ? x_at[i] : ninf, i);
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const uint64_t key = lane < all_hits ? list.keys[lane] : 0;
        int rank = 0;
        for (int j = 0; j < all_hits; j++) rank += list.keys[j] > key;
        if (lane < all_hits && rank < a.beams) to[rank] = key;
        return;
    }
    // many equal values, or a few lanes with large ones: the values above the
    // bound, and in order of their places the first k at it
    n = 0;
    int ties = 0;
    for (int u = 0; u < U; u++) {
        const int i = (u * kWave + lane) * 4;
        uint64_t eq[4];
        int rank = ties;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float y = first + i + e < a.vocab ? x_at[first + i + e] : ninf;
            const uint64_t gt = __builtin_amdgcn_ballot_w64(y > bound), below = (1ull << lane) - 1;
            eq[e] = __builtin_amdgcn_ballot_w64(y == bound);
            if (y > bound) {
                const int at = n + (int)__popcll(gt & below);
                list.apart.value[at] = y;
                list.apart.place[at] = (uint16_t)(i + e);
            }
            n += (int)__popcll(gt);
            rank += (int)__popcll(eq[e] & below);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (eq[e] >> lane & 1) {
                if (rank < a.beams) list.apart.tie[rank] = (uint16_t)(i + e);
                rank++;
            }
            ties += (int)__popcll(eq[e]);
        }
        ties = min(ties, a.beams);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int i0 = 0; i0 < n; i0 += kWave) {
        const int i = min(i0 + lane, n - 1);
        const uint64_t key = beam_key(list.apart.value[i], list.apart.place[i]);
        int rank = 0;
        for (int j = 0; j < n; j++) rank += beam_key(list.apart.value[j], list.apart.place[j]) > key;
        if (i0 + lane < n && rank < a.beams) to[rank] = beam_key(list.apart.value[i], first + list.apart.place[i]);
    }
    if (n + lane < a.beams) to[n + lane] = lane < ties ? beam_key(bound, first + list.apart.tie[lane]) : 0;
}

// A workgroup a group, a wave a beam.  A row's records are sorted lists, one a
// lane: its k best are k times the largest of the lanes' heads.  K: beams, at most.
template <int K>
__global__ __launch_bounds__(K *kWave) void beam_best_kernel(BeamArgs a)
{
    __shared__ uint64_t lists[K][K * kBeamUnits];
    __shared__ double total[K * K];
    __shared__ int ranks[K * K];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int k = a.beams, row = blockIdx.x * k + wave, n = a.units * k;
    // (every load at once)
    const auto keys = make_rsrc(a.keys + (size_t)row * n, (uint32_t)n * 8u);
    u32x2 words[K];
    const float2 s = lane < a.units ? a.sums[(size_t)row * a.units + lane] : make_float2(-__builtin_inff(), 0.0f);
    const float score = a.scores[row];
#pragma unroll
    for (int i = 0; i < K; i++)
        if (i < k) words[i] = __builtin_amdgcn_raw_buffer_load_b64(keys, (i * kWave + lane) * 8, 0, 0);
#pragma unroll
    for (int i = 0; i < K; i++)
        if (i < k) {
            const uint64_t key = (uint64_t)words[i].y << 32 | words[i].x;
            lists[wave][i * kWave + lane] = beam_place(key) < a.vocab ? key : 0;  // (none, or behind the row's end)
        }
    if (lane < k) ranks[wave * k + lane] = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    // the row's distribution (units: a lane each)
    const bool odd = __builtin_amdgcn_ballot_w64(s.x != s.x) != 0;
    const float top = lanes_max(s.x);
    double part = s.y > 0.0f ? (double)s.y * exp((double)s.x - (double)top) : 0.0;
    for (int by = 1; by < kWave; by *= 2) part += __shfl_xor(part, by);
    // (no distribution, or a score that is not finite: every continuation counts -inf)
    const bool ok = !odd && top > -__builtin_inff() && finite_bits(abs_bits(score));
    const double lse = (double)top + log(part);
    uint64_t mine = 0;  // lane i: the row's i-th best
    if (ok) {
        const uint64_t *list = lists[wave] + lane * k;
        int at = 1;
        uint64_t head = lane < a.units ? list[0] : 0, next = lane < a.units && k > 1 ? list[1] : 0;
        for (int i = 0; i < k; i++) {
            const unsigned high = wave_max_u32((unsigned)(head >> 32));
            bool won = (unsigned)(head >> 32) == high;
            const uint64_t who = __builtin_amdgcn_ballot_w64(won);
            if (who & (who - 1)) {  // (equal values: the lowest token)
                const unsigned low = wave_max_u32(won ? (unsigned)head : 0u);
                won = won && (unsigned)head == low;
            }
            const int winner = __builtin_ctzll(__builtin_amdgcn_ballot_w64(won));
            const unsigned first = (unsigned)__builtin_amdgcn_readlane((int)head, winner);
            if (lane == i) mine = (uint64_t)high << 32 | first;
            if (lane == winner) {
                head = next;
                at++;
                next = at < k ? list[at] : 0;
            }
        }
    } else if (lane < k) {
        mine = beam_key(-__builtin_inff(), lane);
    }
    if (lane < k) {
        // (key 0: the row has no k tokens; behind everything)
        total[wave * k + lane] = mine == 0 ? __builtin_nan("") : ok ? (double)beam_value(mine) - lse + (double)score : -__builtin_inf();
    }
    __syncthreads();
    // each total's rank among the group's: against the wave's row's
    double row_total[K];
#pragma unroll
    for (int j = 0; j < K; j++)
        if (j < k) row_total[j] = total[wave * k + j];
    for (int i = lane; i < k * k; i += kWave) {
        const double x = total[i];
        int rank = 0;
#pragma unroll
        for (int j = 0; j < K; j++)
            if (j < k) rank += row_total[j] > x || (row_total[j] == x && wave * k + j < i);
        if (rank) atomicAdd(&ranks[i], rank);
    }
    __syncthreads();
    const int i = wave * k + lane;
    if (lane < k) {
        const double x = total[i];
        const int rank = ranks[i];
        if (x == x && rank < k) {
            const int to = blockIdx.x * k + rank;
            a.parent[to] = row;
            a.token[to] = beam_place(mine);
            a.best[to] = (float)x;
        }
    }
}

}  // namespace leap
