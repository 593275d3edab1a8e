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
// latency, and for long sequences also by the bounds' bytes: of 11.4 us for
// 2048 pages and 8 KV heads of 128 (17 MB) 4.4 go to the scores, 1.5 to the
// arrival, 2.7 to the selection.
#pragma once

#include "paged_attention.hpp"

namespace leap {

constexpr int kSelectWaves = 8, kSelectThreads = kSelectWaves * kWave;
constexpr int kSelectPages = 16384;                         // pages of a sequence, at most
constexpr int kSelectKeys = kSelectPages / kSelectThreads;  // keys of a thread
constexpr int kSelectBins = 2048;
constexpr int kSelectPart = 8;                              // workgroups that count in one place
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
    int *part_counters;       // [group][parts], kCtrStride apart: likewise
    int width, keep, picked_keep, n_pages;
    int n_seq, max_pos, n_heads, n_kv_heads, group, rows_log2;
    int units, parts;         // workgroups of a group, and parts of kSelectPart of them
    FastDiv by_kv_heads, by_units;
};

__device__ __forceinline__ uint64_t score_key(double x)
{
    if (x != x) return ~0ull;
    const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ uint64_t min_u64(uint64_t a, uint64_t b) { return a < b ? a : b; }

struct SelectLds {
    int bins[kSelectBins];
    unsigned ends[2][kSelectWaves];
    int scan[kSelectWaves];
    uint16_t order[kSelectPages];
    int last, found, above, inside;
};

// The `need` largest of n > need keys, up to KEYS a thread, into the list (and
// picked) in order of the pages; the bins are zero.
template <int KEYS>
__device__ __forceinline__ void select_pages(SelectLds &sh, const uint64_t *keys, const int *table, int *list, int *picked, int n, int need, int tid)
{
    const int lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int per = (n + kSelectThreads - 1) / kSelectThreads;  // a thread's keys, in order of the pages
    uint64_t mine[KEYS];
    const auto r = make_rsrc(keys, (uint32_t)n * 8u);
    u32x2 w[KEYS];
#pragma unroll
    for (int i = 0; i < KEYS; i++) {
        // (behind a thread's or all keys: 0, which is no key)
        w[i] = __builtin_amdgcn_raw_buffer_load_b64(r, i < per ? (tid * per + i) * 8 : n * 8, 0, kSc1);
    }
    unsigned most = 0, least_inv = 0;  // of the keys' upper halves
#pragma unroll
    for (int i = 0; i < KEYS; i++) {
        mine[i] = (uint64_t)w[i].y << 32 | w[i].x;
        most = max(most, w[i].y);
        least_inv = max(least_inv, mine[i] ? ~w[i].y : 0u);
    }
    most = wave_max_u32(most);
    least_inv = wave_max_u32(least_inv);
    if (lane == 0) {
        sh.ends[0][wave] = least_inv;
        sh.ends[1][wave] = most;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSelectWaves; w++) {
        least_inv = max(least_inv, sh.ends[0][w]);
        most = max(most, sh.ends[1][w]);
    }
    uint64_t lo = (uint64_t)~least_inv << 32, hi = (uint64_t)most << 32 | 0xffffffffu;
    // the need-th largest: the range that it lies in, narrowed by a
    // histogram of 2048 bins at a time
    int left = need;
    for (int round = 0; round < 6; round++) {  // (64 bits, 11 at a time)
        const uint64_t range = hi - lo;
        const int shift = max(0, 53 - (range ? (int)__builtin_clzll(range) : 64));
#pragma unroll
        for (int i = 0; i < KEYS; i++) {
            if (mine[i] >= lo && mine[i] <= hi) atomicAdd(&sh.bins[(int)((mine[i] - lo) >> shift)], 1);
        }
        __syncthreads();
        // bins from the top, four a thread
        constexpr int B = kSelectBins / kSelectThreads;
        int x[B], sum = 0;
#pragma unroll
        for (int i = 0; i < B; i++) {
            x[i] = sh.bins[kSelectBins - 1 - (tid * B + i)];
            sh.bins[kSelectBins - 1 - (tid * B + i)] = 0;
            sum += x[i];
        }
        const int upto = wave_scan_add(sum);
        if (lane == kWave - 1) sh.scan[wave] = upto;
        __syncthreads();
        int before = upto - sum;
#pragma unroll
        for (int w = 0; w < kSelectWaves; w++) before += w < wave ? sh.scan[w] : 0;
#pragma unroll
        for (int i = 0; i < B; i++) {
            if (before < left && before + x[i] >= left) {
                sh.found = kSelectBins - 1 - (tid * B + i);
                sh.above = before;
                sh.inside = x[i];
            }
            before += x[i];
        }
        __syncthreads();
        left -= sh.above;
        lo += (uint64_t)sh.found << shift;
        if (sh.inside == left || shift == 0) break;
        hi = lo + min_u64(hi - lo, (1ull << shift) - 1);
    }
    // every key from the least taken on, or so many of those equal to it
    const uint64_t least = lo;
    const int ties = sh.inside == left ? 0x7fffffff : left;
    // the chosen ones in order of the pages
    auto scan_all = [&](int x) {
        const int upto = wave_scan_add(x);
        __syncthreads();
        if (lane == kWave - 1) sh.scan[wave] = upto;
        __syncthreads();
        int before = upto - x;
#pragma unroll
        for (int w = 0; w < kSelectWaves; w++) before += w < wave ? sh.scan[w] : 0;
        return before;
    };
    int equal = 0;
    if (ties != 0x7fffffff) {
#pragma unroll
        for (int i = 0; i < KEYS; i++) {
            equal += mine[i] == least;
        }
        equal = scan_all(equal);
    }
    unsigned take = 0;
#pragma unroll
    for (int i = 0; i < KEYS; i++) {
        if (ties == 0x7fffffff ? mine[i] >= least : mine[i] > least || (mine[i] == least && equal++ < ties)) take |= 1u << i;
    }
    int to = scan_all(__popc(take));
    while (take) {
        sh.order[to++] = (uint16_t)(tid * per + __builtin_ctz(take));
        take &= take - 1;
    }
    __syncthreads();
    for (int i = tid; i < need; i += kSelectThreads) {
        const int at = sh.order[i];
        list[i] = table[at];
        if (picked) picked[i] = at;
    }
}

template <int HD>
__global__ __launch_bounds__(kSelectThreads) void page_select_kernel(SelectArgs a)
{
    constexpr int D = HD / 64;  // float4 words of a bound that a lane holds
    __shared__ float4 q[kPagedHeads][HD / 4];
    __shared__ SelectLds sh;
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
        constexpr int S = kPagesAStep / 4, kStep = kSelectWaves * kPagesAStep;
        const int c = lane & 15, per = (n + a.units - 1) / a.units, end = min(n, (unit + 1) * per);
        int p0 = unit * per + wave * kPagesAStep, pages[S];
        bool here[S];
        float4 lo_next[S][D], hi_next[S][D];
        const auto names = make_rsrc(table, (uint32_t)n * 4u);
        auto look = [&](int p0) {
#pragma unroll
            for (int s = 0; s < S; s++)
                pages[s] = (int)__builtin_amdgcn_raw_buffer_load_b32(names, (p0 + 4 * s + (lane >> 4)) * 4, 0, 0);
        };
        auto fetch = [&](int p0) {
#pragma unroll
            for (int s = 0; s < S; s++) {
                here[s] = p0 + 4 * s + (lane >> 4) < end && (unsigned)pages[s] < (unsigned)a.n_pages;
                const float4 *b = reinterpret_cast<const float4 *>(a.bounds) +
                                  ((size_t)(here[s] ? pages[s] : 0) * a.n_kv_heads + kvh) * (HD / 2);
#pragma unroll
                for (int d = 0; d < D; d++) {
                    lo_next[s][d] = b[16 * d + c];
                    hi_next[s][d] = b[HD / 4 + 16 * d + c];
                }
            }
        };
        look(p0);
        for (int i = tid; i < a.group * (HD / 4); i += kSelectThreads) {
            const int head = i / (HD / 4), c = i - head * (HD / 4);
            const float4 x = reinterpret_cast<const float4 *>(a.q + ((size_t)seq * a.n_heads + kvh * a.group) * HD)[i];
            q[head][c] = rope4(x, a.rope[(size_t)pos * (HD / 4) + c]);
        }
        fetch(p0);
        look(p0 + kStep);
        __syncthreads();
        for (; p0 < end; p0 += kStep) {
            // (the next pages' bounds are on their way while these are added up)
            bool there[S];
            float4 lo[S][D], hi[S][D];
#pragma unroll
            for (int s = 0; s < S; s++) {
                there[s] = here[s];
#pragma unroll
                for (int d = 0; d < D; d++) {
                    lo[s][d] = lo_next[s][d];
                    hi[s][d] = hi_next[s][d];
                }
            }
            if (p0 + kStep < end) {
                fetch(p0 + kStep);
                look(p0 + 2 * kStep);
            }
            __builtin_amdgcn_sched_barrier(0);
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
    for (int i = tid; i < kSelectBins; i += kSelectThreads) sh.bins[i] = 0;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
        // (the one that counts last, and leaves the counter zero)
        auto last_of = [](int *at, int n) {
            if (__hip_atomic_fetch_add(at, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != n - 1) return false;
            __hip_atomic_store(at, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            return true;
        };
        // in eights: 32 workgroups counting in one place wait 3 us for each other
        const int part = unit / kSelectPart;
        sh.last = (a.units == 1 || last_of(a.part_counters + ((size_t)gi * a.parts + part) * kCtrStride,
                                           min(kSelectPart, a.units - part * kSelectPart))) &&
                  (a.parts == 1 || last_of(a.counters + gi, a.parts));
    }
    __syncthreads();
    if (!sh.last) return;
    // (a thread's keys without a branch for each: what is skipped is fetched all the same)
    if (need > 0) {
        if (n <= 4 * kSelectThreads)
            select_pages<4>(sh, keys, table, list, picked, n, need, tid);
        else if (n <= 8 * kSelectThreads)
            select_pages<8>(sh, keys, table, list, picked, n, need, tid);
        else
            select_pages<kSelectKeys>(sh, keys, table, list, picked, n, need, tid);
    }
    if (tid == 0) list[need] = table[n];
    if (picked)
        for (int i = need + tid; i < a.picked_keep; i += kSelectThreads) picked[i] = i == need ? n : -1;
}

}  // namespace leap
