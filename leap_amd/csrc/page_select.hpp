// The pages that a new token attends to, for each KV head, where it attends to
// some of a sequence's pages only: the page of its own row, and of the pages
// before it those with the largest scores; of equal scores the earlier page.
//
// A page's score is the sum over the KV head's q heads of the most that q . k
// can be for keys within the page's bounds, sum_i max(q_i lo_i, q_i hi_i), with
// q rotated (products and sums rounded, as keys are).  It is summed in 64
// bits, so that the choice does not hang on the order of a sum.  A score that
// is not a number comes first, and so does a page that is missing: the step
// then shows it.
//
// One launch: the workgroups of a (sequence, KV head), all on one XCD, score
// its pages, 16 lanes a page, and the last one to arrive selects.  Bound by
// the bounds' bytes for long sequences, else by latency.
#pragma once

#include "paged_attention.hpp"

namespace leap {

constexpr int kSelectWaves = 8, kSelectThreads = kSelectWaves * kWave;
constexpr int kSelectPages = 16384;                         // pages of a sequence, at most
constexpr int kSelectKeys = kSelectPages / kSelectThreads;  // keys of a thread
constexpr int kSelectBins = 2048;
constexpr int kPagesAStep = 8;                              // pages of a wave at a time

struct SelectArgs {
    const float *q;
    const float4 *rope;
    const int *pos, *table;
    const float *bounds;      // the layer's
    uint64_t *keys;           // [group][width]
    int *lists;               // [group][keep]
    int *picked;              // [group][picked_keep], or NULL
    int *counters;            // [group], zero between launches
    int width, keep, picked_keep, n_pages;
    int n_seq, max_pos, n_heads, n_kv_heads, group, rows_log2;
    int units;                // workgroups of a group
    FastDiv by_kv_heads, by_units;
};

__device__ __forceinline__ uint64_t score_key(double x)
{
    if (x != x) return ~0ull;
    const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ uint64_t min_u64(uint64_t a, uint64_t b) { return a < b ? a : b; }
__device__ __forceinline__ uint64_t max_u64(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t shfl_xor_u64(uint64_t x, int by)
{
    return (uint64_t)(unsigned)__shfl_xor((int)(x >> 32), by) << 32 | (unsigned)__shfl_xor((int)x, by);
}

template <int HD>
__global__ __launch_bounds__(kSelectThreads) void page_select_kernel(SelectArgs a)
{
    constexpr int D = HD / 64;  // float4 words of a bound that a lane holds
    __shared__ float4 q[kPagedHeads][HD / 4];
    __shared__ int bins[kSelectBins];
    __shared__ uint64_t ends[2][kSelectWaves];
    __shared__ int scan[kSelectWaves];
    __shared__ int last, found, above, inside;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int local = blockIdx.x / kXcds, gl = (int)fast_div((uint32_t)local, a.by_units);
    const int unit = local - gl * a.units, gi = gl * kXcds + (blockIdx.x & (kXcds - 1));
    if (gi >= a.n_seq * a.n_kv_heads) return;
    const int seq = (int)fast_div((uint32_t)gi, a.by_kv_heads), kvh = gi - seq * a.n_kv_heads;
    const int pos = a.pos[seq];
    int *picked = a.picked ? a.picked + (size_t)gi * a.picked_keep : nullptr;
    if (pos < 0 || pos > a.max_pos) {
        if (unit == 0 && picked)
            for (int i = tid; i < a.picked_keep; i += kSelectThreads) picked[i] = -1;
        return;
    }
    const int n = pos >> a.rows_log2, need = a.keep - 1;  // pages before the row's, and how many of them
    const int *table = a.table + (size_t)seq * a.width;
    int *list = a.lists + (size_t)gi * a.keep;
    if (n <= need) {
        if (unit == 0) {
            for (int i = tid; i <= n; i += kSelectThreads) list[i] = table[i];
            if (picked)
                for (int i = tid; i < a.picked_keep; i += kSelectThreads) picked[i] = i <= n ? i : -1;
        }
        return;
    }
    uint64_t *keys = a.keys + (size_t)gi * a.width;
    if (need > 0) {
        // ---- scores ----
        for (int i = tid; i < a.group * (HD / 4); i += kSelectThreads) {
            const int head = i / (HD / 4), c = i - head * (HD / 4);
            const float4 x = reinterpret_cast<const float4 *>(a.q + ((size_t)seq * a.n_heads + kvh * a.group) * HD)[i];
            q[head][c] = rope4(x, a.rope[(size_t)pos * (HD / 4) + c]);
        }
        __syncthreads();
        const int c = lane & 15, per = (n + a.units - 1) / a.units, end = min(n, (unit + 1) * per);
        for (int p0 = unit * per + wave * kPagesAStep; p0 < end; p0 += kSelectWaves * kPagesAStep) {
            constexpr int S = kPagesAStep / 4;
            float4 lo[S][D], hi[S][D];
            bool there[S];
#pragma unroll
            for (int s = 0; s < S; s++) {
                const int at = p0 + 4 * s + (lane >> 4), page = at < end ? table[at] : -1;
                there[s] = (unsigned)page < (unsigned)a.n_pages;
                const float4 *b = reinterpret_cast<const float4 *>(a.bounds) +
                                  ((size_t)(there[s] ? page : 0) * a.n_kv_heads + kvh) * (HD / 2);
#pragma unroll
                for (int d = 0; d < D; d++) {
                    lo[s][d] = b[16 * d + c];
                    hi[s][d] = b[HD / 4 + 16 * d + c];
                }
            }
            double sum[S];
#pragma unroll
            for (int s = 0; s < S; s++) sum[s] = 0.0;
            for (int head = 0; head < a.group; head++)
#pragma unroll
                for (int d = 0; d < D; d++) {
                    const float4 x = q[head][16 * d + c];
                    auto add = [&](double &to, float x, float lo, float hi) {
                        // (products of two floats are exact)
                        to = __builtin_fma((double)x, (double)(x > 0.0f ? hi : lo), to);
                    };
#pragma unroll
                    for (int s = 0; s < S; s++) {
                        add(sum[s], x.x, lo[s][d].x, hi[s][d].x);
                        add(sum[s], x.y, lo[s][d].y, hi[s][d].y);
                        add(sum[s], x.z, lo[s][d].z, hi[s][d].z);
                        add(sum[s], x.w, lo[s][d].w, hi[s][d].w);
                    }
                }
#pragma unroll
            for (int s = 0; s < S; s++) {
#pragma unroll
                for (int by = 1; by < 16; by *= 2) sum[s] += __shfl_xor(sum[s], by);
                const int at = p0 + 4 * s + (lane >> 4);
                if (c == 0 && at < end) keys[at] = there[s] ? score_key(sum[s]) : ~0ull;
            }
        }
    }
    // ---- the last workgroup of the group to arrive selects ----
    // (in one XCD's L2: the stores have drained to it, and the loads miss in L1)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
        const int before = __hip_atomic_fetch_add(a.counters + gi, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = before == a.units - 1;
        if (before == a.units - 1) __hip_atomic_store(a.counters + gi, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last) return;
    uint64_t least = ~0ull;  // the least key taken, and how many of those that have it
    int ties = 0;
    uint64_t mine[kSelectKeys];
    const int per = (n + kSelectThreads - 1) / kSelectThreads;  // a thread's keys, in order of the pages
    if (need > 0) {
        const auto r = make_rsrc(keys, (uint32_t)n * 8u);
        uint64_t lo = ~0ull, hi = 0;
#pragma unroll
        for (int i = 0; i < kSelectKeys; i++) {
            const int at = tid * per + i;
            if (i < per && at < n) {
                const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(r, at * 8, 0, kSc1);
                mine[i] = (uint64_t)w.y << 32 | w.x;
                lo = min_u64(lo, mine[i]);
                hi = max_u64(hi, mine[i]);
            }
        }
        for (int by = 1; by < kWave; by *= 2) {
            lo = min_u64(lo, shfl_xor_u64(lo, by));
            hi = max_u64(hi, shfl_xor_u64(hi, by));
        }
        if (lane == 0) {
            ends[0][wave] = lo;
            ends[1][wave] = hi;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kSelectWaves; w++) {
            lo = min_u64(lo, ends[0][w]);
            hi = max_u64(hi, ends[1][w]);
        }
        // the need-th largest: the range that it lies in, narrowed by a
        // histogram of 2048 bins at a time
        int left = need;
        for (int round = 0; round < 6; round++) {  // (64 bits, 11 at a time)
            const uint64_t range = hi - lo;
            const int shift = max(0, 53 - (range ? (int)__builtin_clzll(range) : 64));
            for (int i = tid; i < kSelectBins; i += kSelectThreads) bins[i] = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kSelectKeys; i++) {
                if (i < per && tid * per + i < n && mine[i] >= lo && mine[i] <= hi) atomicAdd(&bins[(int)((mine[i] - lo) >> shift)], 1);
            }
            __syncthreads();
            // bins from the top, four a thread
            constexpr int B = kSelectBins / kSelectThreads;
            int x[B], sum = 0;
#pragma unroll
            for (int i = 0; i < B; i++) {
                x[i] = bins[kSelectBins - 1 - (tid * B + i)];
                sum += x[i];
            }
            const int upto = wave_scan_add(sum);
            if (lane == kWave - 1) scan[wave] = upto;
            __syncthreads();
            int before = upto - sum;
#pragma unroll
            for (int w = 0; w < kSelectWaves; w++) before += w < wave ? scan[w] : 0;
#pragma unroll
            for (int i = 0; i < B; i++) {
                if (before < left && before + x[i] >= left) {
                    found = kSelectBins - 1 - (tid * B + i);
                    above = before;
                    inside = x[i];
                }
                before += x[i];
            }
            __syncthreads();
            left -= above;
            lo += (uint64_t)found << shift;
            if (inside == left || shift == 0) break;
            hi = lo + min_u64(hi - lo, (1ull << shift) - 1);
        }
        least = lo;
        ties = left;
        if (inside == left) ties = 0x7fffffff;  // (every key from lo on)
    }
    // the chosen ones in order of the pages
    auto scan_all = [&](int x) {
        const int upto = wave_scan_add(x);
        __syncthreads();
        if (lane == kWave - 1) scan[wave] = upto;
        __syncthreads();
        int before = upto - x;
#pragma unroll
        for (int w = 0; w < kSelectWaves; w++) before += w < wave ? scan[w] : 0;
        return before;
    };
    if (need > 0) {
        int equal = 0;
        if (ties != 0x7fffffff) {
#pragma unroll
            for (int i = 0; i < kSelectKeys; i++) {
                if (i < per) equal += tid * per + i < n && mine[i] == least;
            }
            equal = scan_all(equal);
        }
        unsigned take = 0;
#pragma unroll
        for (int i = 0; i < kSelectKeys; i++) {
            if (i < per && tid * per + i < n && (ties == 0x7fffffff ? mine[i] >= least : mine[i] > least || (mine[i] == least && equal++ < ties))) take |= 1u << i;
        }
        int to = scan_all(__popc(take));
        while (take) {
            const int at = tid * per + __builtin_ctz(take);
            take &= take - 1;
            list[to] = table[at];
            if (picked) picked[to] = at;
            to++;
        }
    }
    if (tid == 0) list[need] = table[n];
    if (picked)
        for (int i = need + tid; i < a.picked_keep; i += kSelectThreads) picked[i] = i == need ? n : -1;
}

}  // namespace leap
