// The pages of a pool: which sequence holds which (tables, counts of
// references), and moving their contents.
//
// table [sequence][width] names a sequence's pages in order (-1: none),
// refs [page] counts the tables that name a page, bit p % 32 of
// free_bits [p / 32] is set where refs is 0, and whole [sequence] counts a
// sequence's pages ahead of the first that it lacks, so that a step learns
// with its position whether a page is missing.  The calls below are the only
// ones that change them.  Numbers are given by a rule that does not depend on
// timing: the lowest free page first, to the first sequence's first page first.
//
// All are bound by latency (a few dependent passes over a few KB: fork's two
// launches 2.3 and 2.6 us for 4 sequences and 4.6 for 64, compact's plan 7.0 for a
// pool of 489 pages); what copies pages is bound by memory (507 MB moved in 104 us, 4.9
// TB/s, where a large copy reaches 5.2).
#pragma once

#include "paged_attention.hpp"

namespace leap {

constexpr int kPlanThreads = 1024;   // the kernels that plan are one workgroup each
constexpr int kPlanWaves = kPlanThreads / kWave;

struct PagesArgs {
    int *table, *refs;
    unsigned *free_bits;
    int *whole;                   // [sequence]
    int *asked, *last;            // [page], 0 and -1 between launches
    int *item;                    // [sequence][width]: scratch (fork: the new tables)
    int *prefix;                  // [sequence + 1]: scratch (fork: the new `whole`)
    int *ids;                     // [page]: scratch (free pages in order; compact: where a page went)
    int2 *copies;                 // [page]: from, to
    int *n_copies;                // [2]: how many copies; pages in use before compact
    const int *parent, *rows;     // fork
    const int *begin, *end;       // reserve
    int *status;                  // reserve: or NULL
    int *count;                   // compact: or NULL
    int n_seq, max_batch, width, n_pages, seq_len, rows_log2;
};

// Inclusive sum over a workgroup of kPlanThreads, and the total; sh: kPlanWaves ints.
__device__ __forceinline__ int block_scan(int x, int *sh, int tid, int *total)
{
    const int lane = tid & (kWave - 1), wave = tid / kWave;
    const int upto = wave_scan_add(x);
    __syncthreads();  // (sh is free)
    if (lane == kWave - 1) sh[wave] = upto;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; w++) {
        const int v = sh[w];
        if (w < wave) before += v;
        all += v;
    }
    *total = all;
    return before + upto;
}
__device__ __forceinline__ int load_now(const int *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void store_now(int *p, int x) { __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The workgroup's stores in sight of its loads, which go past L1.
__device__ __forceinline__ void plan_sync()
{
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// put(i, page) of the pages from first to end whose bit is set (want_free) or
// clear, in ascending order, i < most; returns how many there are, or a number
// that is not below most.  first_word: word first / 32 + tid, loaded ahead.
__device__ __forceinline__ unsigned word_of(const unsigned *bits, int w, int end) { return w < (end + 31) / 32 ? bits[w] : 0u; }
template <class Put>
__device__ __forceinline__ int list_pages(const unsigned *bits, bool want_free, int first, int end, int most, unsigned first_word, int *sh, int tid, Put put)
{
    int found = 0;
    const int words = (end + 31) / 32;
    for (int w0 = first / 32; w0 < words; w0 += kPlanThreads) {
        const int w = w0 + tid;
        unsigned x = 0;
        if (w < words) {
            x = w0 == first / 32 ? first_word : bits[w];
            if (!want_free) x = ~x;
            if (w == first / 32) x &= ~0u << (first & 31);
            if (w == end / 32) x &= (1u << (end & 31)) - 1u;
        }
        int total;
        int at = found + block_scan(__popc(x), sh, tid, &total) - __popc(x);
        while (x && at < most) {
            put(at++, 32 * w + __builtin_ctz(x));
            x &= x - 1;
        }
        found += total;
        if (found >= most) break;
    }
    return found;
}

// What reserve needs to bring `whole` up to date for a sequence that gets the
// pages [first, end): loaded before the table changes, of entries that stay.
struct Whole {
    int seq, first, end, now, next;  // now: whole; next: the page behind the range (-1: none)
};
__device__ __forceinline__ Whole whole_load(const PagesArgs &a, int seq, int first, int end, int now)
{
    Whole w{seq, first, end, now, -1};
    if (end > first && end < a.width) w.next = a.table[(size_t)seq * a.width + end];
    return w;
}
// By all lanes of a wave.  Where the range closes a gap ahead of pages that
// were there, the wave looks for the next one, 64 entries at a time.
__device__ __forceinline__ void whole_store(const PagesArgs &a, const Whole &w, int lane)
{
    const bool grows = w.end > w.first && w.first <= w.now && w.now < w.end;
    if (grows && w.next < 0) a.whole[w.seq] = w.end;
    for (uint64_t left = __builtin_amdgcn_ballot_w64(grows && w.next >= 0); left; left &= left - 1) {
        const int from = __builtin_ctzll(left), seq = __builtin_amdgcn_readlane(w.seq, from);
        uint64_t gap = 0;
        int at = __builtin_amdgcn_readlane(w.end, from);
        for (; !gap; at += gap ? __builtin_ctzll(gap) : kWave)
            gap = __builtin_amdgcn_ballot_w64(at + lane >= a.width || a.table[(size_t)seq * a.width + at + lane] < 0);
        if (lane == 0) a.whole[seq] = at;
    }
}

// reserve_kernel's way for up to 1024 sequences and items (a step's: one item a
// sequence): LDS and registers, an item a thread.
constexpr int kBadRange = (int)0x80000000u;
constexpr int kAskedSlots = 2 * kPlanThreads;
struct ReserveFew {
    int first[kPlanThreads];      // items ahead of each sequence's
    int base[kPlanThreads];       // a sequence's page of item f: base + f
    int ids[kPlanThreads];        // free pages, in order
    int page[kAskedSlots], asked[kAskedSlots], last[kAskedSlots];  // shared pages: how many ask, and the last of them
};
// The page's slot, put there if it is new.
__device__ __forceinline__ int asked_slot(int *pages, int page)
{
    unsigned at = ((unsigned)page * 2654435761u) >> 21;  // (of 2048; a page in 1024 at most: an empty slot is always left)
    static_assert(kAskedSlots == 2048, "slots");
    for (;; at = (at + 1) & (kAskedSlots - 1)) {
        const int there = atomicCAS(&pages[at], -1, page);
        if (there == page || there == -1) return (int)at;
    }
}
__device__ __forceinline__ void reserve_few(const PagesArgs &a, ReserveFew &l, int *sh, int *copies, int items, const Whole &whole, int tid, int e_nomem)
{
    const unsigned word = word_of(a.free_bits, tid, a.n_pages);
    int seq = 0, page = -1, refs = 0;
    size_t at = 0;
    const bool mine = tid < items;
    if (mine) {
        int hi = a.n_seq - 1;  // the last sequence that begins at f or before: the only such that has items
        while (seq < hi) {
            const int mid = (seq + hi + 1) / 2;
            if (l.first[mid] <= tid)
                seq = mid;
            else
                hi = mid - 1;
        }
        at = (size_t)seq * a.width + l.base[seq] + tid;
        page = a.table[at];
        if (page >= 0) refs = a.refs[page];
    }
    bool take = mine && page < 0;
    if (__syncthreads_or(refs > 1)) {
        for (int i = tid; i < kAskedSlots; i += kPlanThreads) {
            l.page[i] = -1;
            l.asked[i] = 0;
            l.last[i] = -1;
        }
        __syncthreads();
        int slot = 0;
        if (refs > 1) {
            slot = asked_slot(l.page, page);
            atomicAdd(&l.asked[slot], 1);
            atomicMax(&l.last[slot], seq);
        }
        __syncthreads();
        if (refs > 1) take = !(l.asked[slot] == refs && l.last[slot] == seq);
    }
    int need;
    const int rank = block_scan(take, sh, tid, &need) - 1;
    bool granted = true;
    if (need > 0) {
        const int n_free = list_pages(a.free_bits, true, 0, a.n_pages, need, word, sh, tid, [&](int i, int page) { l.ids[i] = page; });
        __syncthreads();
        granted = n_free >= need;
        if (!granted) {
            if (a.status && tid < a.n_seq && l.base[tid] != kBadRange) a.status[tid] = e_nomem;
        } else if (take) {
            const int to = l.ids[rank];
            if (page >= 0) {
                __hip_atomic_fetch_add(a.refs + page, -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                a.copies[atomicAdd(copies, 1)] = make_int2(page, to);
            }
            a.refs[to] = 1;
            __hip_atomic_fetch_and(a.free_bits + (to >> 5), ~(1u << (to & 31)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            a.table[at] = to;
        }
    }
    if (granted) whole_store(a, whole, tid & (kWave - 1));
    __syncthreads();
    if (tid == 0) a.n_copies[0] = *copies;
}

// Rows [begin, end) of each sequence will be written: their pages are there
// afterwards and named by no other table.  A missing page is a free one, a
// shared one a copy, but the last of the sequences that share a page keeps it
// where all of them ask for it.  If the pool has too few free pages nothing
// changes and every status is -ENOMEM; a sequence with a bad range is left
// out, -EINVAL.  Items: the (sequence, page) pairs asked for, in order.
//
// Bound by its chain of trips to memory: ranges, tables, counts, results.  With
// up to 1024 items 7.8 us for 64 sequences that share pages and 4.4 for 4,
// where the passes over memory below take 11.6 and 6.5.  Beyond that each item
// looks for its sequence three times: 4 sequences of 512 pages 47 us, 32 254, 64
// 500.
__global__ __launch_bounds__(kPlanThreads) void reserve_kernel(PagesArgs a, int e_inval, int e_nomem)
{
    __shared__ int sh[kPlanWaves];
    __shared__ int copies;
    __shared__ ReserveFew few;
    const int tid = threadIdx.x, R = 1 << a.rows_log2;
    if (tid == 0) copies = 0;
    // items ahead of each sequence's
    int items = 0;
    const bool in_lds = a.n_seq <= kPlanThreads;
    Whole whole{0, 0, 0, 0, -1};  // (of sequence tid: where all are in LDS)
    for (int i0 = 0; i0 < a.n_seq; i0 += kPlanThreads) {
        const int i = i0 + tid;
        int n = 0, b = 0;
        bool ok = false;
        if (i < a.n_seq) {
            const int e = a.end[i], now = a.whole[i];
            b = a.begin[i];
            ok = b >= 0 && b <= e && e <= a.seq_len;
            if (ok && b < e) {
                n = ((e + R - 1) >> a.rows_log2) - (b >> a.rows_log2);
                if (in_lds) whole = whole_load(a, i, b >> a.rows_log2, (e + R - 1) >> a.rows_log2, now);
            }
            if (a.status) a.status[i] = ok ? 0 : e_inval;
        }
        int total;
        const int upto = items + block_scan(n, sh, tid, &total);
        if (i < a.n_seq) {
            if (in_lds) {
                few.first[i] = upto - n;
                few.base[i] = ok ? (b >> a.rows_log2) - (upto - n) : kBadRange;
            } else {
                store_now(a.prefix + i + 1, upto);
            }
        }
        items += total;
    }
    __syncthreads();  // (few.first: either way the next wave's is read)
    if (in_lds && items <= kPlanThreads) {
        reserve_few(a, few, sh, &copies, items, whole, tid, e_nomem);
        return;
    }
    if (in_lds && tid < a.n_seq) store_now(a.prefix + tid + 1, tid + 1 < a.n_seq ? few.first[tid + 1] : items);
    if (tid == 0) store_now(a.prefix, 0);
    plan_sync();
    // an item's sequence and place in the table
    auto place = [&](int f, int *seq) {
        int lo = 0, hi = a.n_seq - 1;  // the last sequence that begins at f or before, and has items
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (load_now(a.prefix + mid) <= f)
                lo = mid;
            else
                hi = mid - 1;
        }
        *seq = lo;
        return (size_t)lo * a.width + (a.begin[lo] >> a.rows_log2) + (f - load_now(a.prefix + lo));
    };
    // who asks for shared pages
    bool shared = false;
    for (int f = tid; f < items; f += kPlanThreads) {
        int i;
        const int page = a.table[place(f, &i)];
        if (page >= 0 && a.refs[page] > 1) {
            shared = true;
            __hip_atomic_fetch_add(a.asked + page, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_fetch_max(a.last + page, i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    shared = __syncthreads_or(shared);
    if (shared) plan_sync();
    // which items take a free page, and which of them in order
    int need = 0;
    bool granted = true;
    for (int f0 = 0; f0 < items; f0 += kPlanThreads) {
        const int f = f0 + tid;
        bool take = false;
        if (f < items) {
            int i;
            const int page = a.table[place(f, &i)];
            take = page < 0;
            if (page >= 0) {
                const int refs = a.refs[page];
                take = refs > 1 && !(load_now(a.asked + page) == refs && load_now(a.last + page) == i);
            }
        }
        int total;
        const int upto = need + block_scan(take, sh, tid, &total);
        if (f < items) a.item[f] = take ? upto - 1 : -1;  // (read back by the thread that writes it)
        need += total;
    }
    if (need > 0) {
        const int n_free = list_pages(a.free_bits, true, 0, a.n_pages, need, word_of(a.free_bits, tid, a.n_pages), sh, tid,
                                      [&](int i, int page) { store_now(a.ids + i, page); });
        plan_sync();
        granted = n_free >= need;
        if (!granted) {
            if (a.status)
                for (int i = tid; i < a.n_seq; i += kPlanThreads)
                    if (a.begin[i] >= 0 && a.begin[i] <= a.end[i] && a.end[i] <= a.seq_len) a.status[i] = e_nomem;
        }
    }
    for (int f = tid; f < items; f += kPlanThreads) {
        int i;
        const size_t at = place(f, &i);
        const int page = a.table[at], rank = a.item[f];
        if (granted && rank >= 0) {
            const int to = load_now(a.ids + rank);
            if (page >= 0) {
                __hip_atomic_fetch_add(a.refs + page, -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                a.copies[atomicAdd(&copies, 1)] = make_int2(page, to);
            }
            a.refs[to] = 1;
            __hip_atomic_fetch_and(a.free_bits + (to >> 5), ~(1u << (to & 31)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            a.table[at] = to;
        }
        if (shared && page >= 0) {
            store_now(a.asked + page, 0);
            store_now(a.last + page, -1);
        }
    }
    if (granted)
        for (int i0 = 0; i0 < a.n_seq; i0 += kPlanThreads) {
            const int i = i0 + tid;
            if (!in_lds) {
                whole = Whole{0, 0, 0, 0, -1};
                if (i < a.n_seq) {
                    const int b = a.begin[i], e = a.end[i];
                    if (b >= 0 && b < e && e <= a.seq_len) whole = whole_load(a, i, b >> a.rows_log2, (e + R - 1) >> a.rows_log2, a.whole[i]);
                }
            }
            whole_store(a, whole, tid & (kWave - 1));
        }
    __syncthreads();
    if (tid == 0) a.n_copies[0] = copies;
}

// New tables: sequence i takes the pages of the first rows[i] rows of
// parent[i] (NULL: of its own), as the tables were before the call; a parent
// or a number of rows out of range leaves it as it is.  Two launches: the new
// names are counted before the old ones are dropped, so that no page is free
// in between.
__global__ __launch_bounds__(256) void fork_gather_kernel(PagesArgs a)
{
    const int i = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
    if (j >= a.width) return;
    const int from = a.parent ? a.parent[i] : i, rows = a.rows[i];
    const int old = a.table[(size_t)i * a.width + j];
    const bool ok = from >= 0 && from < a.max_batch && rows >= 0 && rows <= a.seq_len;
    const int whole = a.whole[ok ? from : i];
    int page = old;
    if (ok) page = (long long)j << a.rows_log2 < rows ? a.table[(size_t)from * a.width + j] : -1;
    if (j == 0) a.prefix[i] = ok ? min(whole, (rows + (1 << a.rows_log2) - 1) >> a.rows_log2) : whole;
    a.item[(size_t)i * a.width + j] = page;
    if (page >= 0 && page != old) __hip_atomic_fetch_add(a.refs + page, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__global__ __launch_bounds__(256) void fork_drop_kernel(PagesArgs a)
{
    const int i = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
    if (j >= a.width) return;
    const size_t at = (size_t)i * a.width + j;
    const int old = a.table[at], page = a.item[at], whole = a.prefix[i];
    if (j == 0) a.whole[i] = whole;
    if (page == old) return;
    a.table[at] = page;
    if (old >= 0 && __hip_atomic_fetch_add(a.refs + old, -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 1)
        __hip_atomic_fetch_or(a.free_bits + (old >> 5), 1u << (old & 31), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The pages in use move down until none is free below one of them: the i-th
// page in use from number n on (n of them are in use) goes to the i-th free
// page below n.  page_copy_kernel moves what they hold and renames them in
// the tables.
__global__ __launch_bounds__(kPlanThreads) void compact_kernel(PagesArgs a)
{
    __shared__ int sh[kPlanWaves];
    const int tid = threadIdx.x, words = (a.n_pages + 31) / 32;
    int n_free = 0;
    for (int w0 = 0; w0 < words; w0 += kPlanThreads) {
        int total;
        (void)block_scan(w0 + tid < words ? __popc(a.free_bits[w0 + tid]) : 0, sh, tid, &total);
        n_free += total;
    }
    const int used = a.n_pages - n_free;
    int *copies = reinterpret_cast<int *>(a.copies);
    const int moves = list_pages(a.free_bits, true, 0, used, a.n_pages, word_of(a.free_bits, tid, used), sh, tid,
                                 [&](int i, int page) { store_now(copies + 2 * i + 1, page); });
    list_pages(a.free_bits, false, used, a.n_pages, moves, word_of(a.free_bits, used / 32 + tid, a.n_pages), sh, tid,
               [&](int i, int page) { store_now(copies + 2 * i, page); });
    plan_sync();
    for (int i = tid; i < moves; i += kPlanThreads) {
        const int from = load_now(copies + 2 * i), to = load_now(copies + 2 * i + 1);
        a.refs[to] = a.refs[from];
        a.refs[from] = 0;
        a.ids[from] = to;
    }
    for (int w = tid; w < words; w += kPlanThreads) {
        unsigned x = 32 * w + 32 <= a.n_pages ? ~0u : (1u << (a.n_pages & 31)) - 1u;
        if (32 * w + 32 <= used)
            x = 0;
        else if (32 * w < used)
            x &= ~0u << (used & 31);
        a.free_bits[w] = x;
    }
    if (tid == 0) {
        a.n_copies[0] = moves;
        a.n_copies[1] = used;
        if (a.count) *a.count = used;
    }
}

// What a plan's copied pages hold, in every layer: the five arrays of a page
// one after the other, in pieces of 16 KiB.  compact: the workgroups from
// copy_wgs on rename the pages in the tables instead.
struct CopyArgs {
    char *at[5];                   // k, v, ks, vs, bounds: the first layer's first page
    long long layer[5];            // bytes between layers
    unsigned bytes[5];             // of a page
    const int2 *copies;
    const int *n_copies;
    int n_layers, pieces;          // pieces of a page of one layer
    int copy_wgs, rename;
    int *table;                    // compact: [entries]
    const int *ids;
    long long entries;
};
constexpr unsigned kPiece = 16384;
__global__ __launch_bounds__(256) void page_copy_kernel(CopyArgs a)
{
    const int tid = threadIdx.x, n = a.n_copies[0];
    if (a.rename && (int)blockIdx.x >= a.copy_wgs) {
        const int used = a.n_copies[1];
        const long long step = (long long)(gridDim.x - a.copy_wgs) * 256;
        for (long long i = (long long)(blockIdx.x - a.copy_wgs) * 256 + tid; i < a.entries; i += step) {
            const int page = a.table[i];
            if (page >= used) a.table[i] = a.ids[page];
        }
        return;
    }
    const long long items = (long long)n * a.n_layers * a.pieces;
    for (long long i = blockIdx.x; i < items; i += a.copy_wgs) {
        long long cl = i / a.pieces;
        const unsigned piece = (unsigned)(i - cl * a.pieces);
        const int c = (int)(cl / a.n_layers), layer = (int)(cl - (long long)c * a.n_layers);
        const int2 move = a.copies[c];
        f32x4 x[4];
        char *to[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            unsigned off = piece * kPiece + (unsigned)(u * 256 + tid) * 16u;
            to[u] = nullptr;
#pragma unroll
            for (int k = 0; k < 5; k++) {
                if (!to[u] && off < a.bytes[k]) {
                    char *base = a.at[k] + layer * a.layer[k] + off;
                    x[u] = *reinterpret_cast<const f32x4 *>(base + (size_t)move.x * a.bytes[k]);
                    to[u] = base + (size_t)move.y * a.bytes[k];
                } else if (!to[u]) {
                    off -= a.bytes[k];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (to[u]) *reinterpret_cast<f32x4 *>(to[u]) = x[u];
    }
}

}  // namespace leap
