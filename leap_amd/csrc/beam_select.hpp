// The selection of a beam search: of all continuations (beam, token) of a
// group of beams, the best by score[beam] + log_softmax(logits[beam])[token].
//
// Two launches.  beam_rows_kernel reads the logits once: a wave takes up to
// 4096 of a row, keeps them in registers, and leaves the row's maximum and sum
// of exponentials over them and their `beams` best, in order.  The k-th
// largest of the lanes' maxima bounds the k-th largest of all from below, so
// that few values are looked at one by one.  beam_best_kernel joins a group's
// records: a wave a row, then all rows' best against each other, in 64 bits.
// Bound by the logits' bytes, or for few rows by latency.
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

__device__ __forceinline__ unsigned wave_max_u32(unsigned x) { return rows4_bits(dpp_max16(x)); }

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

// The first k of n keys in LDS, best first, into to[0 .. k) (0: none).
__device__ __forceinline__ void best_keys(const uint64_t *list, int n, int k, uint64_t *to, int lane)
{
    for (int i0 = 0; i0 < n; i0 += kWave) {
        const uint64_t mine = i0 + lane < n ? list[i0 + lane] : 0;
        int rank = 0;
        for (int j = 0; j < n; j++) rank += list[j] > mine;
        if (i0 + lane < n && rank < k) to[rank] = mine;
    }
    for (int i = n + lane; i < k; i += kWave) to[i] = 0;
}

// U words of four logits a lane.
template <int U>
__global__ __launch_bounds__(256) void beam_rows_kernel(BeamArgs a)
{
    constexpr int kList = (kBeamMax - 1) * 4 * U + kBeamMax;  // values above the bound (in at most k - 1 lanes), and k at it
    __shared__ uint64_t lists[4][kList];
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const long long at = (long long)blockIdx.x * 4 + wave;
    const int row = (int)(at / a.units), unit = (int)(at - (long long)row * a.units);
    if (row >= a.rows) return;
    const float *x_at = a.logits + row * a.stride;
    const int first = unit * (U * 4 * kWave);
    const float ninf = -__builtin_inff();
    float x[U][4];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int i = first + (u * kWave + lane) * 4;
        if (i + 4 <= a.vocab) {
            f32x4 y;
            __builtin_memcpy(&y, x_at + i, 16);  // (rows need not be aligned)
#pragma unroll
            for (int e = 0; e < 4; e++) x[u][e] = y[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) x[u][e] = i + e < a.vocab ? x_at[i + e] : ninf;
        }
    }
    float top = ninf;
    bool odd = false;  // NaN or +inf
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            odd |= !(x[u][e] < __builtin_inff());
            top = fmaxf(top, x[u][e]);
        }
    odd = __builtin_amdgcn_ballot_w64(odd) != 0;
    const unsigned mine = (unsigned)(beam_key(top, 0) >> 32);
    const float all = lanes_max(top);
    float sum = 0.0f;
    if (all > ninf && !odd) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) sum += fast_exp2((x[u][e] - all) * 1.44269504088896341f);
    }
    sum = lanes_sum(sum);
    if (lane == 0) a.sums[at] = make_float2(odd ? __uint_as_float(0x7fc00000u) : all, sum);
    uint64_t *to = a.keys + at * a.beams;
    if (odd) return;  // (its row has no distribution: beam_best_kernel does not look at these)
    // the values above the bound, and in order of their places the first k at it
    const unsigned b = kth_largest(mine, a.beams);
    const float bound = beam_value((uint64_t)b << 32);
    uint64_t *list = lists[wave];
    int n = 0, ties = 0;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int i = first + (u * kWave + lane) * 4;
        const float w = fmaxf(fmaxf(x[u][0], x[u][1]), fmaxf(x[u][2], x[u][3]));
        if (__builtin_amdgcn_ballot_w64(w >= bound) == 0) continue;
        uint64_t eq[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint64_t gt = __builtin_amdgcn_ballot_w64(x[u][e] > bound);
            eq[e] = __builtin_amdgcn_ballot_w64(x[u][e] == bound);
            if (x[u][e] > bound) list[n + (int)__popcll(gt & ((1ull << lane) - 1))] = beam_key(x[u][e], i + e);
            n += (int)__popcll(gt);
        }
        if (ties < a.beams) {
            int rank = ties;
#pragma unroll
            for (int e = 0; e < 4; e++) rank += (int)__popcll(eq[e] & ((1ull << lane) - 1));
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (x[u][e] == bound) {
                    if (rank < a.beams) list[kList - 1 - rank] = beam_key(x[u][e], i + e);
                    rank++;
                }
#pragma unroll
            for (int e = 0; e < 4; e++) ties += (int)__popcll(eq[e]);
        }
    }
    ties = min(ties, a.beams);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    // (together: the ties behind the others)
    uint64_t tie = 0;
    if (lane < ties) tie = list[kList - 1 - lane];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (lane < ties) list[n + lane] = tie;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    best_keys(list, n + ties, a.beams, to, lane);
}

// A workgroup a group, a wave a beam.
__global__ __launch_bounds__(kBeamMax *kWave) void beam_best_kernel(BeamArgs a)
{
    __shared__ uint64_t lists[kBeamMax][kBeamMax * kBeamMax];  // (k - 1 lanes' kBeamMax keys, and k)
    __shared__ uint64_t best[kBeamMax][kBeamMax];
    __shared__ double lse[kBeamMax], total[kBeamMax * kBeamMax];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int k = a.beams, row = blockIdx.x * k + wave;
    const double ninf = -__builtin_inf();
    if (wave < k) {
        // the row's distribution (units: a lane each)
        const float2 s = lane < a.units ? a.sums[(size_t)row * a.units + lane] : make_float2(-__builtin_inff(), 0.0f);
        const bool odd = __builtin_amdgcn_ballot_w64(s.x != s.x) != 0;
        const float top = lanes_max(s.x), score = a.scores[row];
        double part = s.y > 0.0f ? (double)s.y * exp((double)s.x - (double)top) : 0.0;
        for (int by = 1; by < kWave; by *= 2) part += __shfl_xor(part, by);
        // (no distribution, or a score that is not finite: every continuation counts -inf)
        const bool ok = !odd && top > -__builtin_inff() && finite_bits(abs_bits(score));
        if (lane == 0) lse[wave] = ok ? (double)top + log(part) : __builtin_inf();
        // its k best
        if (ok) {
            const int n = a.units * k;
            const uint64_t *keys = a.keys + (size_t)row * n;
            uint64_t mine[kBeamMax], most = 0;
#pragma unroll
            for (int i = 0; i < kBeamMax; i++) {
                const int at = i * kWave + lane;
                mine[i] = at < n ? keys[at] : 0;
                if (beam_place(mine[i]) >= a.vocab) mine[i] = 0;  // (none, or behind the row's end)
                most = mine[i] > most ? mine[i] : most;
            }
            // those of values above the bound, in at most k - 1 lanes, and the first k at it
            const unsigned bound = kth_largest((unsigned)(most >> 32), k);
            int count = 0;
#pragma unroll
            for (int pass = 0; pass < 2; pass++) {
                const int end = pass ? count + k : kBeamMax * kBeamMax;
#pragma unroll
                for (int i = 0; i < kBeamMax; i++) {
                    const unsigned v = (unsigned)(mine[i] >> 32);
                    const bool in = mine[i] != 0 && (pass ? v == bound : v > bound);
                    const uint64_t who = __builtin_amdgcn_ballot_w64(in);
                    const int to = count + (int)__popcll(who & ((1ull << lane) - 1));
                    if (in && to < end) lists[wave][to] = mine[i];
                    count = min(count + (int)__popcll(who), end);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            best_keys(lists[wave], count, k, best[wave], lane);
        } else if (lane < k) {
            best[wave][lane] = beam_key(-__builtin_inff(), lane);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (lane < k) {
            const uint64_t key = best[wave][lane];
            // (key 0: the row has no k tokens; behind everything)
            total[wave * k + lane] = key == 0 ? __builtin_nan("") : ok ? (double)beam_value(key) - lse[wave] + (double)score : ninf;
        }
    }
    __syncthreads();
    for (int i = tid; i < k * k; i += blockDim.x) {
        const double mine = total[i];
        if (mine != mine) continue;
        int rank = 0;
        for (int j = 0; j < k * k; j++) {
            const double y = total[j];
            rank += y > mine || (y == mine && j < i);
        }
        if (rank < k) {
            const int to = blockIdx.x * k + rank;
            a.parent[to] = blockIdx.x * k + i / k;
            a.token[to] = beam_place(best[i / k][i % k]);
            a.best[to] = (float)mine;
        }
    }
}

}  // namespace leap
