// C-ABI of caches of pages (include/leap_hip_attention.h): argument checks,
// the pool and its tables in device memory, and what launches are cut into.
// Device side: paged_attention.hpp, page_ops.hpp, page_rows.hpp,
// page_select.hpp, beam_select.hpp.
#include "leap_hip_attention.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cerrno>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <new>
#include <string>
#include <vector>

#include "beam_select.hpp"
#include "host_util.hpp"
#include "kernels.hpp"
#include "page_ops.hpp"

extern "C" void leap_rope_table_host(int seq_len, int head_size, float theta, float *cos_tab, float *sin_tab);

struct leap_hip_attention_pages {
    leap_hip_attention_pages_config cfg{};
    int n_local = 0, kv_dim = 0, q_dim = 0, group = 0, width = 0, rows_log2 = 0;
    int n_cu = 256;
    bool q8 = false;
    // bytes of a page of one layer: k, v, ks, vs, bounds; and the arrays
    size_t page_bytes[5] = {};
    char *pool[5] = {};
    float4 *rope = nullptr;
    int *table = nullptr, *refs = nullptr;
    unsigned *free_bits = nullptr;
    int *whole = nullptr, *asked = nullptr, *last = nullptr, *item = nullptr, *prefix = nullptr, *ids = nullptr, *n_copies = nullptr;
    int2 *copies = nullptr;
    // the step's records and counters; the sparse step's keys, lists and counters
    float *ws_o = nullptr, *ws_lse = nullptr;
    int *counters = nullptr;
    uint64_t *keys = nullptr;
    int *lists = nullptr, *select_counters = nullptr;
    // the beam selection's records (its first call)
    uint64_t *beam_keys = nullptr;
    float2 *beam_sums = nullptr;
    // the host-pointer calls' staging (the tables' calls' from the start, else grown)
    char *staging = nullptr;
    size_t staging_bytes = 0;
    hipStream_t stream = nullptr;
    std::string err;
};

using namespace leap_kernels;
using leap_host::launch_k;

namespace {

thread_local char g_pages_error[512];

int set_err(leap_hip_attention_pages *p, int code, const char *fmt, ...)
{
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    if (p)
        p->err = buf;
    else
        std::memcpy(g_pages_error, buf, sizeof buf);
    return code;
}

// (the thread's sticky code is read, so that no later query reports it)
#define HIP_TRY(p, call)                                                                      \
    do {                                                                                      \
        hipError_t e_ = (call);                                                               \
        if (e_ != hipSuccess) {                                                               \
            (void)hipGetLastError();                                                          \
            return set_err((p), e_ == hipErrorOutOfMemory ? -ENOMEM : -EIO, "%s: %s", #call, \
                           hipGetErrorString(e_));                                            \
        }                                                                                     \
    } while (0)

constexpr int kMaxPages = 1 << 26;
constexpr int kMaxRows = 1 << 24;
// Head records and counters that a handle holds (32 MiB of outputs at head_dim
// 128): a launch that would leave more takes longer runs.
constexpr size_t kRecords = 65536;
constexpr size_t kCounters = 4096;
// fp32 rows that a host transfer stages at a time.
constexpr size_t kStagingBytes = size_t(8) << 20;
// A group that streams this much runs on all XCDs where there are fewer groups
// than XCDs.
constexpr long long kSpreadBytes = 4ll << 20;

long long round_up(long long x, int q) { return (x + q - 1) / q * q; }
bool aligned(const void *p, unsigned by) { return reinterpret_cast<uintptr_t>(p) % by == 0; }

int check_layer(leap_hip_attention_pages *p, int layer)
{
    const auto &m = p->cfg.model;
    if (layer < m.layer_begin || layer >= m.layer_end)
        return set_err(p, -EINVAL, "layer %d outside the held range [%d, %d)", layer, m.layer_begin, m.layer_end);
    return 0;
}
int check_seqs(leap_hip_attention_pages *p, int n_seq)
{
    if (n_seq <= 0 || n_seq > p->cfg.model.max_batch)
        return set_err(p, -EINVAL, "n_seq %d outside [1, %d]", n_seq, p->cfg.model.max_batch);
    return 0;
}

template <typename T>
T *layer_at(const leap_hip_attention_pages *p, int array, int layer)
{
    return reinterpret_cast<T *>(p->pool[array] + (size_t)(layer - p->cfg.model.layer_begin) * p->cfg.n_pages * p->page_bytes[array]);
}

int staging(leap_hip_attention_pages *p, size_t bytes)
{
    if (bytes <= p->staging_bytes) return 0;
    char *q = nullptr;
    HIP_TRY(p, hipMalloc(&q, bytes));
    if (p->staging) (void)hipFree(p->staging);
    p->staging = q;
    p->staging_bytes = bytes;
    return 0;
}

// ---- the step ------------------------------------------------------------------

struct StepPlan {
    int chunk, splits;
    bool spread, flat;
    long long wgs;
};
// total: rows of all sequences; longest: of one, both along what is attended to.
//
// Uniform launches cut every group into runs of the same length.  Their time,
// past a constant, is near the larger of what memory and a run take, and the
// merge: a tile of a wave takes 1.65 us (8 bits 2.4) from its loads to its
// products, four waves at a time, tiles come in at 6.8 TB/s over the card (8
// bits: an eighth slower with one workgroup a CU; fp32 a tenth over long runs
// of one sequence), 1 us of them within the constant, and records take 2 us
// and 0.03 for each.  (us, 32/8/128, runs of 4, 8, 16, 32 tiles: fp32, one
// sequence of 4096 11.2, 11.2, 13.6, 19.9, of 8192 -, 17.8, 16.7, 22.6; 12 of
// 4096 -, 73, 72, 64.6; 8 bits, one of 4096 10.4, 13.2, of 16384 16.5, 15.3.)
// What it leaves out: a workgroup's start, and that rounds of workgroups
// overlap.  So equal lengths whose groups do not divide by the CUs get the
// shortest runs, which stream less: sequences of 4096, 32/8/128, fp32 32 166,
// 33 210, 40 211, 45 281, 48 251; 8 bits 57, 70, 76, 91, 78.
//
// Batches of unequal lengths with a group for every XCD run flat once they have
// 16 tiles a CU (uniform : flat; 32/8/128 fp32, 8 sequences of up to 500 9.8 :
// 11.3, 16 of up to 1000 22.5 : 21.0, 32 of up to 7300 180 : 163, 64/8/128 16
// of up to 7300 124 : 108; 8 bits, 32 of up to 8192 73 : 68; equal lengths, 16
// of 8192 160 : 162, 8 bits 32 of 8192 100 : 110).  Two workgroups a CU: 8 bits
// need both (one: 84), fp32 takes as long with one.  A lane holds one group of
// its XCD, so that more than 512 groups stay uniform: of up to 4096, 32/32/128,
// 16 sequences (flat) 162, 17 213, 20 298; 8 bits 62, 86, 104.  Without a count
// of rows the lengths are taken as unequal.
StepPlan step_plan(const leap_hip_attention_pages *p, int n_seq, int longest, long long total)
{
    const int n_kv = p->cfg.model.n_kv_heads, hd = p->cfg.model.head_dim, tk = leap::paged_tile(hd, p->q8);
    const long long groups = (long long)n_seq * n_kv, items = (groups + leap::kXcds - 1) / leap::kXcds;
    const long long mean = (total + n_seq - 1) / n_seq;
    const long long tiles_mean = (mean + tk - 1) / tk, tiles_max = (longest + tk - 1) / tk;
    const long long group_bytes = mean * (p->q8 ? 2ll * (hd + 4) : 8ll * hd);
    const bool few = groups < leap::kXcds && group_bytes < kSpreadBytes;  // on as many XCDs as groups
    const double cus = few ? p->n_cu * groups / (double)leap::kXcds : p->n_cu;
    const double tile_us = (p->q8 ? hd / 128.0 : 1.0) * 0.0024, run_us = p->q8 ? 2.4 : 1.65;
    StepPlan s{};
    double best = 0;
    for (int n = 1; n <= leap::kPagedSplits && n <= tiles_max; n++) {
        // (a tile for every wave, or as many)
        const long long chunk = n == 1 ? tiles_max : round_up((tiles_max + n - 1) / n, leap::kPagedWaves);
        if (n > 1 && (chunk == s.chunk || (size_t)groups * n * p->group > kRecords || (size_t)groups > kCounters)) continue;
        const double wgs = groups * std::ceil((double)tiles_mean / chunk);
        const double rate = wgs < cus ? 0.9 : wgs > cus ? 1.0 : p->q8 ? 1.125 : 1.03;
        const double memory = std::ceil(wgs / cus) * chunk * tile_us * p->n_cu * rate - 1.0;
        const double run = std::ceil(chunk / (double)leap::kPagedWaves) * run_us;
        const double us = std::max(memory, run) + (n > 1 ? 2.0 + 0.03 * n : 0.0);
        if (n == 1 || us < best) {
            best = us;
            s.chunk = (int)chunk;
            s.splits = (int)((tiles_max + chunk - 1) / chunk);
        }
    }
    const long long flat_wgs = 2ll * p->n_cu;
    const bool equal = total == (long long)n_seq * longest;
    const bool fits = items <= leap::kWave && (size_t)(leap::kXcds * items + flat_wgs) * p->group <= kRecords &&
                      (size_t)groups <= kCounters && flat_wgs <= (long long)leap::kXcds * leap::kPagedSplits;
    if (n_seq > 1 && groups >= leap::kXcds && !equal && groups * tiles_mean >= 16ll * p->n_cu && fits)
        return StepPlan{1, (int)items, false, true, flat_wgs};
    s.spread = s.splits > 1 && groups < leap::kXcds && !few;
    s.wgs = s.spread ? groups * s.splits : items * leap::kXcds * s.splits;
    return s;
}

// keep 0: over all pages; else the lists hold keep pages a group.
int launch_step(leap_hip_attention_pages *p, int layer, int n_seq, const int *pos, int max_pos, long long total, int keep,
                const float *q, const float *k, const float *v, float *out, hipStream_t stream)
{
    const auto &m = p->cfg.model;
    const int longest = keep ? std::min(max_pos + 1, keep << p->rows_log2) : max_pos + 1;
    const StepPlan s = step_plan(p, n_seq, longest, keep ? (long long)n_seq * longest : total);
    const PagedKernels fn = pick_paged(m.head_dim, p->group, p->q8);
    leap::PagedArgs a{};
    a.q = q;
    a.k_new = k;
    a.v_new = v;
    a.out = out;
    a.k = layer_at<void>(p, 0, layer);
    a.v = layer_at<void>(p, 1, layer);
    if (p->q8) {
        a.ks = layer_at<float>(p, 2, layer);
        a.vs = layer_at<float>(p, 3, layer);
    }
    if (p->cfg.bounds) a.bounds = layer_at<float>(p, 4, layer);
    a.rope = p->rope;
    a.pos = pos;
    a.table = p->table;
    a.refs = p->refs;
    a.whole = p->whole;
    a.lists = p->lists;
    a.ws_o = p->ws_o;
    a.ws_lse = p->ws_lse;
    a.counters = p->counters;
    a.width = p->width;
    a.keep = keep;
    a.n_pages = p->cfg.n_pages;
    a.n_seq = n_seq;
    a.max_pos = max_pos;
    a.n_heads = m.n_heads;
    a.n_kv_heads = m.n_kv_heads;
    a.group = p->group;
    a.rows_log2 = p->rows_log2;
    a.chunk = s.chunk;
    a.splits = s.splits;
    a.blocks = (longest + 15) / 16;
    a.spread = s.spread;
    a.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)m.head_dim));
    a.by_kv_heads = leap::make_fastdiv((uint32_t)m.n_kv_heads);
    a.by_splits = leap::make_fastdiv((uint32_t)s.splits);
    a.by_chunk = leap::make_fastdiv((uint32_t)s.chunk);
    a.by_groups = leap::make_fastdiv((uint32_t)(n_seq * m.n_kv_heads));
    if (s.wgs > 0x7fffffffLL) return set_err(p, -EINVAL, "%lld workgroups in one launch", s.wgs);
    HIP_TRY(p, launch_k(s.flat ? fn.flat : fn.attention, dim3((unsigned)s.wgs), dim3(leap::kPagedWaves * leap::kWave), stream, a));
    if (s.spread) HIP_TRY(p, launch_k(fn.merge, dim3((unsigned)(n_seq * m.n_kv_heads)), dim3(256), stream, a));
    return 0;
}

// A counter for each group, and one for each part of the groups' workgroups:
// two workgroups a CU at most where a group has more than one.
size_t select_counters(const leap_hip_attention_pages *p)
{
    const long long groups = (long long)p->cfg.model.max_batch * p->cfg.model.n_kv_heads;
    const long long parts = 2ll * p->n_cu / leap::kSelectPart + p->n_cu;
    return (size_t)(round_up(groups, leap::kCtrStride) + parts * leap::kCtrStride);
}

int launch_select(leap_hip_attention_pages *p, int layer, int n_seq, const int *pos, int max_pos, int keep, int picked_keep,
                  const float *q, int *picked, hipStream_t stream)
{
    const auto &m = p->cfg.model;
    const long long groups = (long long)n_seq * m.n_kv_heads;
    const int pages = max_pos >> p->rows_log2;  // scored, at most
    leap::SelectArgs a{};
    a.q = q;
    a.rope = p->rope;
    a.pos = pos;
    a.table = p->table;
    a.bounds = layer_at<float>(p, 4, layer);
    a.keys = p->keys;
    a.lists = p->lists;
    a.picked = picked;
    a.counters = p->select_counters;
    a.part_counters = p->select_counters + round_up((long long)p->cfg.model.max_batch * m.n_kv_heads, leap::kCtrStride);
    a.width = p->width;
    a.keep = keep;
    a.picked_keep = picked_keep;
    a.n_pages = p->cfg.n_pages;
    a.n_seq = n_seq;
    a.max_pos = max_pos;
    a.n_heads = m.n_heads;
    a.n_kv_heads = m.n_kv_heads;
    a.group = p->group;
    a.rows_log2 = p->rows_log2;
    // a step of a workgroup's waves at least, two workgroups a CU at most
    const long long most = std::max<long long>(1, 2ll * p->n_cu / groups);
    const long long step = leap::kSelectWaves * leap::kPagesAStep;
    a.units = (int)std::max<long long>(1, std::min(most, (pages + step - 1) / step));
    a.parts = (a.units + leap::kSelectPart - 1) / leap::kSelectPart;
    a.by_kv_heads = leap::make_fastdiv((uint32_t)m.n_kv_heads);
    a.by_units = leap::make_fastdiv((uint32_t)a.units);
    const long long wgs = (groups + leap::kXcds - 1) / leap::kXcds * leap::kXcds * a.units;
    if (wgs > 0x7fffffffLL) return set_err(p, -EINVAL, "%lld workgroups in one launch", wgs);
    HIP_TRY(p, launch_k(pick_paged(m.head_dim, p->group, p->q8).select, dim3((unsigned)wgs), dim3(leap::kSelectThreads), stream, a));
    return 0;
}

int step_checks(leap_hip_attention_pages *p, int layer, int n_seq, const int *pos, int max_pos, long long total, const float *q,
                const float *k, const float *v, const float *out)
{
    if (int rc = check_layer(p, layer)) return rc;
    if (int rc = check_seqs(p, n_seq)) return rc;
    if (max_pos < 0 || max_pos >= p->cfg.model.seq_len)
        return set_err(p, -EINVAL, "max_pos %d outside [0, %d)", max_pos, p->cfg.model.seq_len);
    if (total < 0 || total > (long long)n_seq * (max_pos + 1))
        return set_err(p, -EINVAL, "total_rows %lld outside [0, %lld]", total, (long long)n_seq * (max_pos + 1));
    if (!pos || !q || !k || !v || !out) return set_err(p, -EINVAL, "NULL buffer");
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16) || !aligned(pos, 4))
        return set_err(p, -EINVAL, "q, k_new, v_new and out must be 16-byte aligned, pos 4-byte aligned");
    return 0;
}

// ---- tables ----------------------------------------------------------------------

leap::PagesArgs pages_args(const leap_hip_attention_pages *p, int n_seq)
{
    leap::PagesArgs a{};
    a.table = p->table;
    a.refs = p->refs;
    a.free_bits = p->free_bits;
    a.whole = p->whole;
    a.asked = p->asked;
    a.last = p->last;
    a.item = p->item;
    a.prefix = p->prefix;
    a.ids = p->ids;
    a.copies = p->copies;
    a.n_copies = p->n_copies;
    a.n_seq = n_seq;
    a.max_batch = p->cfg.model.max_batch;
    a.width = p->width;
    a.n_pages = p->cfg.n_pages;
    a.seq_len = p->cfg.model.seq_len;
    a.rows_log2 = p->rows_log2;
    return a;
}

// The copies of the plan before, and (rename) the tables after compact.
int launch_copies(leap_hip_attention_pages *p, bool rename, hipStream_t stream)
{
    leap::CopyArgs a{};
    size_t total = 0;
    for (int k = 0; k < 5; k++) {
        a.at[k] = p->pool[k];
        a.layer[k] = (long long)(p->page_bytes[k] * (size_t)p->cfg.n_pages);
        a.bytes[k] = p->pool[k] ? (unsigned)p->page_bytes[k] : 0u;
        total += a.bytes[k];
    }
    a.copies = p->copies;
    a.n_copies = p->n_copies;
    a.n_layers = p->n_local;
    a.pieces = (int)((total + leap::kPiece - 1) / leap::kPiece);
    a.copy_wgs = 8 * p->n_cu;
    a.rename = rename;
    a.table = p->table;
    a.ids = p->ids;
    a.entries = (long long)p->cfg.model.max_batch * p->width;
    const int more = rename ? (int)std::min<long long>(p->n_cu, (a.entries + 255) / 256) : 0;
    HIP_TRY(p, launch_k(leap::page_copy_kernel, dim3((unsigned)(a.copy_wgs + more)), dim3(256), stream, a));
    return 0;
}

int launch_reserve(leap_hip_attention_pages *p, int n_seq, const int *begin, const int *end, int *status, hipStream_t stream)
{
    leap::PagesArgs a = pages_args(p, n_seq);
    a.begin = begin;
    a.end = end;
    a.status = status;
    HIP_TRY(p, launch_k(leap::reserve_kernel, dim3(1), dim3(leap::kPlanThreads), stream, a, -EINVAL, -ENOMEM));
    return launch_copies(p, false, stream);
}

// (checked) ranges in host memory; *status: the device's answer.
int reserve_host(leap_hip_attention_pages *p, int n_seq, const int *begin, const int *end, int *status)
{
    HIP_TRY(p, hipSetDevice(p->cfg.model.device));
    const size_t bytes = (size_t)n_seq * sizeof(int);
    if (int rc = staging(p, 3 * bytes)) return rc;
    int *bd = reinterpret_cast<int *>(p->staging), *ed = bd + n_seq, *sd = ed + n_seq;
    HIP_TRY(p, hipMemcpyAsync(bd, begin, bytes, hipMemcpyHostToDevice, p->stream));
    HIP_TRY(p, hipMemcpyAsync(ed, end, bytes, hipMemcpyHostToDevice, p->stream));
    if (int rc = launch_reserve(p, n_seq, bd, ed, sd, p->stream)) return rc;
    HIP_TRY(p, hipMemcpyAsync(status, sd, sizeof *status, hipMemcpyDeviceToHost, p->stream));  // (one for all)
    HIP_TRY(p, hipStreamSynchronize(p->stream));
    return 0;
}

int launch_fork(leap_hip_attention_pages *p, int n_seq, const int *parent, const int *rows, hipStream_t stream)
{
    leap::PagesArgs a = pages_args(p, n_seq);
    a.parent = parent;
    a.rows = rows;
    const dim3 grid((unsigned)((p->width + 255) / 256), (unsigned)n_seq);
    HIP_TRY(p, launch_k(leap::fork_gather_kernel, grid, dim3(256), stream, a));
    HIP_TRY(p, launch_k(leap::fork_drop_kernel, grid, dim3(256), stream, a));
    return 0;
}

// Every table empty, every page free, the pool and the counters zero.
int clear_all(leap_hip_attention_pages *p)
{
    const size_t entries = (size_t)p->cfg.model.max_batch * p->width, n = (size_t)p->cfg.n_pages;
    HIP_TRY(p, hipMemsetAsync(p->table, 0xff, entries * sizeof(int), p->stream));
    HIP_TRY(p, hipMemsetAsync(p->refs, 0, n * sizeof(int), p->stream));
    HIP_TRY(p, hipMemsetAsync(p->whole, 0, (size_t)p->cfg.model.max_batch * sizeof(int), p->stream));
    HIP_TRY(p, hipMemsetAsync(p->asked, 0, n * sizeof(int), p->stream));
    HIP_TRY(p, hipMemsetAsync(p->last, 0xff, n * sizeof(int), p->stream));
    HIP_TRY(p, hipMemsetAsync(p->free_bits, 0xff, (n / 32) * sizeof(unsigned), p->stream));
    if (n % 32) {
        const unsigned tail = (1u << (n % 32)) - 1u;
        HIP_TRY(p, hipMemcpyAsync(p->free_bits + n / 32, &tail, sizeof tail, hipMemcpyHostToDevice, p->stream));
        HIP_TRY(p, hipStreamSynchronize(p->stream));  // (tail)
    }
    for (int k = 0; k < 5; k++)
        if (p->pool[k]) HIP_TRY(p, hipMemsetAsync(p->pool[k], 0, p->page_bytes[k] * n * p->n_local, p->stream));
    HIP_TRY(p, hipMemsetAsync(p->counters, 0, kCounters * leap::kCtrStride * sizeof(int), p->stream));
    if (p->select_counters)
        HIP_TRY(p, hipMemsetAsync(p->select_counters, 0, select_counters(p) * sizeof(int), p->stream));
    HIP_TRY(p, hipStreamSynchronize(p->stream));
    return 0;
}

// ---- rows ------------------------------------------------------------------------

int rows_checks(leap_hip_attention_pages *p, int seq, int layer, int pos_begin, int pos_end)
{
    if (int rc = check_layer(p, layer)) return rc;
    if (seq < 0 || seq >= p->cfg.model.max_batch)
        return set_err(p, -EINVAL, "seq %d outside [0, %d)", seq, p->cfg.model.max_batch);
    if (pos_begin < 0 || pos_end > p->cfg.model.seq_len || pos_begin > pos_end)
        return set_err(p, -EINVAL, "position range [%d, %d) outside [0, %d)", pos_begin, pos_end, p->cfg.model.seq_len);
    return 0;
}
int launch_rows(leap_hip_attention_pages *p, int seq, int layer, int pos_begin, int n, const float *k_in, const float *v_in,
                float *k_out, float *v_out, hipStream_t stream)
{
    leap::PageRowsArgs a{};
    a.k_in = k_in;
    a.v_in = v_in;
    a.k_out = k_out;
    a.v_out = v_out;
    a.k = layer_at<void>(p, 0, layer);
    a.v = layer_at<void>(p, 1, layer);
    if (p->q8) {
        a.ks = layer_at<float>(p, 2, layer);
        a.vs = layer_at<float>(p, 3, layer);
    }
    a.table = p->table + (size_t)seq * p->width;
    a.refs = p->refs;
    a.n_pages = p->cfg.n_pages;
    a.n_kv_heads = p->cfg.model.n_kv_heads;
    a.rows_log2 = p->rows_log2;
    a.row0 = pos_begin;
    a.n = n;
    const PagedKernels fn = pick_paged(p->cfg.model.head_dim, p->group, p->q8);
    const long long words = (long long)n * p->kv_dim / 4;
    const unsigned grid = (unsigned)std::min<long long>((words + 255) / 256, 16ll * p->n_cu);
    HIP_TRY(p, launch_k(k_in || v_in ? fn.write : fn.read, dim3(grid, 2), dim3(256), stream, a));
    if (k_in && p->cfg.bounds) {
        a.bounds = layer_at<float>(p, 4, layer);
        const long long heads = (long long)(((pos_begin + n - 1) >> p->rows_log2) - (pos_begin >> p->rows_log2) + 1) * a.n_kv_heads;
        HIP_TRY(p, launch_k(fn.bounds, dim3((unsigned)((heads + 3) / 4)), dim3(256), stream, a));
    }
    return 0;
}
int rows_async(leap_hip_attention_pages *p, int seq, int layer, int pos_begin, int pos_end, const float *k_in, const float *v_in,
               float *k_out, float *v_out, void *stream)
{
    if (!p) return -EINVAL;
    if (int rc = rows_checks(p, seq, layer, pos_begin, pos_end)) return rc;
    for (const void *x : {(const void *)k_in, (const void *)v_in, (const void *)k_out, (const void *)v_out})
        if (!aligned(x, 16)) return set_err(p, -EINVAL, "k and v must be 16-byte aligned");
    if (pos_begin == pos_end || (!k_in && !v_in && !k_out && !v_out)) return 0;
    HIP_TRY(p, hipSetDevice(p->cfg.model.device));
    return launch_rows(p, seq, layer, pos_begin, pos_end - pos_begin, k_in, v_in, k_out, v_out, (hipStream_t)stream);
}
// Host rows, staged in pieces.
int rows_host(leap_hip_attention_pages *p, int seq, int layer, int pos_begin, int pos_end, const float *k_in, const float *v_in,
              float *k_out, float *v_out)
{
    if (!p) return -EINVAL;
    if (int rc = rows_checks(p, seq, layer, pos_begin, pos_end)) return rc;
    if (pos_begin == pos_end || (!k_in && !v_in && !k_out && !v_out)) return 0;
    HIP_TRY(p, hipSetDevice(p->cfg.model.device));
    if (k_in || v_in) {
        std::vector<int> table, refs;
        try {
            table.resize((size_t)p->width);
            refs.resize((size_t)p->cfg.n_pages);
        } catch (const std::bad_alloc &) {
            return set_err(p, -ENOMEM, "host allocation failed");
        }
        HIP_TRY(p, hipMemcpyAsync(table.data(), p->table + (size_t)seq * p->width, table.size() * sizeof(int), hipMemcpyDeviceToHost, p->stream));
        HIP_TRY(p, hipMemcpyAsync(refs.data(), p->refs, refs.size() * sizeof(int), hipMemcpyDeviceToHost, p->stream));
        HIP_TRY(p, hipStreamSynchronize(p->stream));
        for (int j = pos_begin >> p->rows_log2; j <= (pos_end - 1) >> p->rows_log2; j++)
            if (table[j] < 0 || refs[table[j]] != 1)
                return set_err(p, -EINVAL, "sequence %d has no page of its own for rows %d and on: reserve them", seq,
                               std::max(pos_begin, j << p->rows_log2));
    }
    const int piece = (int)std::max<size_t>(1, kStagingBytes / (2 * (size_t)p->kv_dim * sizeof(float)));
    const size_t most = (size_t)std::min(piece, pos_end - pos_begin) * p->kv_dim;
    if (int rc = staging(p, 2 * most * sizeof(float))) return rc;
    float *kd = reinterpret_cast<float *>(p->staging), *vd = kd + most;
    for (int at = pos_begin; at < pos_end; at += piece) {
        const int rows = std::min(piece, pos_end - at);
        const size_t off = (size_t)(at - pos_begin) * p->kv_dim, bytes = (size_t)rows * p->kv_dim * sizeof(float);
        if (k_in) HIP_TRY(p, hipMemcpyAsync(kd, k_in + off, bytes, hipMemcpyHostToDevice, p->stream));
        if (v_in) HIP_TRY(p, hipMemcpyAsync(vd, v_in + off, bytes, hipMemcpyHostToDevice, p->stream));
        if (int rc = launch_rows(p, seq, layer, at, rows, k_in ? kd : nullptr, v_in ? vd : nullptr, k_out ? kd : nullptr,
                                 v_out ? vd : nullptr, p->stream))
            return rc;
        if (k_out) HIP_TRY(p, hipMemcpyAsync(k_out + off, kd, bytes, hipMemcpyDeviceToHost, p->stream));
        if (v_out) HIP_TRY(p, hipMemcpyAsync(v_out + off, vd, bytes, hipMemcpyDeviceToHost, p->stream));
    }
    HIP_TRY(p, hipStreamSynchronize(p->stream));
    return 0;
}

int beam_checks(leap_hip_attention_pages *p, int n_groups, int beams, int vocab, const float *logits, long long stride,
                const float *score, const int *parent, const int *token, const float *best)
{
    const int most = p->cfg.model.max_batch;
    if (beams < 1 || beams > leap::kBeamMax) return set_err(p, -EINVAL, "beams %d outside [1, %d]", beams, leap::kBeamMax);
    if (n_groups <= 0 || (long long)n_groups * beams > most)
        return set_err(p, -EINVAL, "%d groups of %d beams: outside [1, %d] beams", n_groups, beams, most);
    if (vocab < beams || vocab > leap::kBeamVocab)
        return set_err(p, -EINVAL, "vocab %d outside [%d, %d]", vocab, beams, leap::kBeamVocab);
    if (stride < vocab) return set_err(p, -EINVAL, "stride %lld is below vocab %d", stride, vocab);
    if (!logits || !score || !parent || !token || !best) return set_err(p, -EINVAL, "NULL buffer");
    if (!aligned(logits, 4) || !aligned(score, 4) || !aligned(parent, 4) || !aligned(token, 4) || !aligned(best, 4))
        return set_err(p, -EINVAL, "buffers must be 4-byte aligned");
    return 0;
}
int launch_beam(leap_hip_attention_pages *p, int n_groups, int beams, int vocab, const float *logits, long long stride,
                const float *score, int *parent, int *token, float *best, hipStream_t stream)
{
    if (!p->beam_keys) {
        hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
        HIP_TRY(p, hipStreamIsCapturing(stream, &cap));
        if (cap != hipStreamCaptureStatusNone)
            return set_err(p, -EINVAL, "a handle's first beam selection allocates its workspace: make one before capturing");
        const size_t records = (size_t)p->cfg.model.max_batch * leap::kBeamUnits;
        float2 *sums = nullptr;
        HIP_TRY(p, hipMalloc(&sums, records * sizeof(float2)));
        if (hipError_t e = hipMalloc(&p->beam_keys, records * leap::kBeamMax * sizeof(uint64_t)); e != hipSuccess) {
            (void)hipGetLastError();
            (void)hipFree(sums);
            p->beam_keys = nullptr;
            return set_err(p, e == hipErrorOutOfMemory ? -ENOMEM : -EIO, "hipMalloc: %s", hipGetErrorString(e));
        }
        p->beam_sums = sums;
    }
    leap::BeamArgs a{};
    a.logits = logits;
    a.scores = score;
    a.stride = stride;
    a.vocab = vocab;
    a.beams = beams;
    a.rows = n_groups * beams;
    // 4 words a lane, or 8, while they fit the records and leave up to 16 waves
    // a CU, else 16 (4 rows of 32000: with 4 words 7.5 us, with 16 9.8; 128 rows
    // 9.8 and 10.6; 128 rows of 65536, 32 waves a CU: 14.6 and 13.4; of 128256,
    // 8 words and 16: 1 row 6.4 and 7.6, 8 rows 10.5 and 11.6, 64 14.0 and 14.4)
    const auto units = [&](int words) { return (vocab + words * 4 * leap::kWave - 1) / (words * 4 * leap::kWave); };
    int words = 4;
    while (words < leap::kBeamWords && (units(words) > leap::kBeamUnits || (long long)a.rows * units(words) > 16 * p->n_cu)) words *= 2;
    a.units = units(words);
    a.keys = p->beam_keys;
    a.sums = p->beam_sums;
    a.parent = parent;
    a.token = token;
    a.best = best;
    const unsigned grid = (unsigned)(((long long)a.rows * a.units + 3) / 4);
    const auto rows = words == 4 ? leap::beam_rows_kernel<4> : words == 8 ? leap::beam_rows_kernel<8> : leap::beam_rows_kernel<leap::kBeamWords>;
    HIP_TRY(p, launch_k(rows, dim3(grid), dim3(256), stream, a));
    const auto join = beams <= 4 ? leap::beam_best_kernel<4> : beams <= 8 ? leap::beam_best_kernel<8> : leap::beam_best_kernel<leap::kBeamMax>;
    HIP_TRY(p, launch_k(join, dim3((unsigned)n_groups), dim3((unsigned)(beams * leap::kWave)), stream, a));
    return 0;
}

}  // namespace

extern "C" {

int leap_hip_attention_pages_create(const leap_hip_attention_pages_config *cfg, leap_hip_attention_pages **out)
{
    if (!out) return set_err(nullptr, -EINVAL, "out is NULL");
    *out = nullptr;
    if (!cfg) return set_err(nullptr, -EINVAL, "cfg is NULL");
    const leap_hip_attention_pages_config c = *cfg;
    const leap_hip_attention_config &m = c.model;
    if (m.n_heads <= 0 || m.n_kv_heads <= 0 || m.n_heads % m.n_kv_heads != 0)
        return set_err(nullptr, -EINVAL, "n_heads %d must be a positive multiple of n_kv_heads %d", m.n_heads, m.n_kv_heads);
    const int group = m.n_heads / m.n_kv_heads;
    if ((m.head_dim != 64 && m.head_dim != 128) || !(group <= 4 || group == 8 || group == 16))
        return set_err(nullptr, -EINVAL, "unsupported head_dim %d with %d q heads per kv head", m.head_dim, group);
    if (m.seq_len <= 0 || m.seq_len > kMaxRows || m.n_layers <= 0 || m.layer_begin < 0 || m.layer_end > m.n_layers ||
        m.layer_begin >= m.layer_end)
        return set_err(nullptr, -EINVAL, "bad layer range [%d, %d) of %d or seq_len %d", m.layer_begin, m.layer_end, m.n_layers, m.seq_len);
    if (m.max_batch <= 0 || m.max_batch > 65535) return set_err(nullptr, -EINVAL, "max_batch %d out of range", m.max_batch);
    if (!(m.rope_theta <= 0.0f || std::isfinite(m.rope_theta))) return set_err(nullptr, -EINVAL, "rope_theta must be finite");
    if (c.page_rows != 16 && c.page_rows != 32 && c.page_rows != 64 && c.page_rows != 128)
        return set_err(nullptr, -EINVAL, "page_rows %d is not 16, 32, 64 or 128", c.page_rows);
    if (c.n_pages < 1 || c.n_pages > kMaxPages) return set_err(nullptr, -EINVAL, "n_pages %d outside [1, %d]", c.n_pages, kMaxPages);
    if ((c.q8 != 0 && c.q8 != 1) || (c.bounds != 0 && c.bounds != 1))
        return set_err(nullptr, -EINVAL, "q8 %d and bounds %d must be 0 or 1", c.q8, c.bounds);
    const int width = (m.seq_len + c.page_rows - 1) / c.page_rows;
    // (a reservation counts the pages asked for in 32 bits)
    if ((long long)m.max_batch * width > 0x7fffffff)
        return set_err(nullptr, -EINVAL, "a table of %d sequences of %d pages is too large", m.max_batch, width);
    if (c.bounds && width > leap::kSelectPages)
        return set_err(nullptr, -EINVAL, "%d pages a sequence: with bounds at most %d", width, leap::kSelectPages);
    // (rows of a page and KV head are 32-bit offsets, records of a group 32-bit bytes)
    if ((long long)c.page_rows * m.n_kv_heads * m.head_dim >= 1 << 26)
        return set_err(nullptr, -EINVAL, "a page of %d rows of %d KV heads is too large", c.page_rows, m.n_kv_heads);

    int ndev = 0;
    if (hipGetDeviceCount(&ndev) != hipSuccess || ndev <= 0) return set_err(nullptr, -ENODEV, "no HIP device");
    if (m.device < 0 || m.device >= ndev) return set_err(nullptr, -EINVAL, "device %d of %d", m.device, ndev);

    leap_hip_attention_pages *p = new (std::nothrow) leap_hip_attention_pages;
    if (!p) return set_err(nullptr, -ENOMEM, "host allocation failed");
    p->cfg = c;
    if (p->cfg.model.rope_theta <= 0.0f) p->cfg.model.rope_theta = 500000.0f;
    p->n_local = m.layer_end - m.layer_begin;
    p->kv_dim = m.n_kv_heads * m.head_dim;
    p->q_dim = m.n_heads * m.head_dim;
    p->group = group;
    p->width = width;
    p->q8 = c.q8 == 1;
    while (1 << p->rows_log2 < c.page_rows) p->rows_log2++;
    const size_t head_rows = (size_t)c.page_rows * m.n_kv_heads;
    p->page_bytes[0] = p->page_bytes[1] = head_rows * m.head_dim * (p->q8 ? 1 : sizeof(float));
    p->page_bytes[2] = p->page_bytes[3] = p->q8 ? head_rows * sizeof(float) : 0;
    p->page_bytes[4] = c.bounds ? (size_t)m.n_kv_heads * 2 * m.head_dim * sizeof(float) : 0;

    auto fail = [&](int rc) {
        std::snprintf(g_pages_error, sizeof g_pages_error, "%s", p->err.c_str());
        leap_hip_attention_pages_destroy(p);
        return rc;
    };
    int rc;
#define CREATE_TRY(call)                                                                     \
    do {                                                                                     \
        if ((rc = [&]() -> int { HIP_TRY(p, call); return 0; }()) != 0) return fail(rc);     \
    } while (0)
    CREATE_TRY(hipSetDevice(m.device));
    CREATE_TRY(hipDeviceGetAttribute(&p->n_cu, hipDeviceAttributeMultiprocessorCount, m.device));
    CREATE_TRY(hipStreamCreate(&p->stream));
    if ((rc = leap_host::check_placement(m.device, 2 * p->n_cu, &p->err)) != 0) return fail(rc);
    // the kernels' code (a launch that loads it cannot be captured)
    for (const void *f : {reinterpret_cast<const void *>(pick_paged(m.head_dim, p->group, p->q8).merge),
                          reinterpret_cast<const void *>(&leap::reserve_kernel)}) {
        hipFuncAttributes attr;
        CREATE_TRY(hipFuncGetAttributes(&attr, f));
    }
    for (int k = 0; k < 5; k++)
        if (p->page_bytes[k]) CREATE_TRY(hipMalloc(&p->pool[k], p->page_bytes[k] * (size_t)c.n_pages * p->n_local));
    const size_t entries = (size_t)m.max_batch * width, n = (size_t)c.n_pages, groups = (size_t)m.max_batch * m.n_kv_heads;
    CREATE_TRY(hipMalloc(&p->table, entries * sizeof(int)));
    CREATE_TRY(hipMalloc(&p->item, entries * sizeof(int)));
    CREATE_TRY(hipMalloc(&p->refs, n * sizeof(int)));
    CREATE_TRY(hipMalloc(&p->whole, (size_t)m.max_batch * sizeof(int)));
    CREATE_TRY(hipMalloc(&p->asked, n * sizeof(int)));
    CREATE_TRY(hipMalloc(&p->last, n * sizeof(int)));
    CREATE_TRY(hipMalloc(&p->ids, n * sizeof(int)));
    CREATE_TRY(hipMalloc(&p->copies, n * sizeof(int2)));
    CREATE_TRY(hipMalloc(&p->free_bits, (n + 31) / 32 * sizeof(unsigned)));
    CREATE_TRY(hipMalloc(&p->prefix, ((size_t)m.max_batch + 1) * sizeof(int)));
    CREATE_TRY(hipMalloc(&p->n_copies, 2 * sizeof(int)));
    CREATE_TRY(hipMalloc(&p->ws_o, kRecords * m.head_dim * sizeof(float)));
    CREATE_TRY(hipMalloc(&p->ws_lse, kRecords * sizeof(float)));
    CREATE_TRY(hipMalloc(&p->counters, kCounters * leap::kCtrStride * sizeof(int)));
    if ((rc = staging(p, 3 * (size_t)m.max_batch * sizeof(int))) != 0) return fail(rc);
    if (c.bounds) {
        CREATE_TRY(hipMalloc(&p->keys, groups * width * sizeof(uint64_t)));
        CREATE_TRY(hipMalloc(&p->lists, groups * width * sizeof(int)));
        CREATE_TRY(hipMalloc(&p->select_counters, select_counters(p) * sizeof(int)));
    }
    const size_t rope_n = (size_t)m.seq_len * (m.head_dim / 2);
    std::vector<float> packed;
    try {
        std::vector<float> cs(rope_n), sn(rope_n);
        packed.resize(2 * rope_n);
        leap_rope_table_host(m.seq_len, m.head_dim, p->cfg.model.rope_theta, cs.data(), sn.data());
        for (size_t i = 0; i < rope_n; i++) {
            packed[2 * i] = cs[i];
            packed[2 * i + 1] = sn[i];
        }
    } catch (const std::bad_alloc &) {
        return fail(set_err(p, -ENOMEM, "host allocation failed"));
    }
    CREATE_TRY(hipMalloc(&p->rope, packed.size() * sizeof(float)));
    CREATE_TRY(hipMemcpyAsync(p->rope, packed.data(), packed.size() * sizeof(float), hipMemcpyHostToDevice, p->stream));
    if ((rc = clear_all(p)) != 0) return fail(rc);
#undef CREATE_TRY
    *out = p;
    return 0;
}

int leap_hip_attention_pages_destroy(leap_hip_attention_pages *p)
{
    if (!p) return 0;
    (void)hipSetDevice(p->cfg.model.device);
    if (p->stream) (void)hipStreamSynchronize(p->stream);
    void *bufs[] = {p->pool[0], p->pool[1], p->pool[2], p->pool[3], p->pool[4], p->rope, p->table, p->item, p->refs, p->whole, p->asked,
                    p->last, p->ids, p->copies, p->free_bits, p->prefix, p->n_copies, p->ws_o, p->ws_lse, p->counters, p->keys,
                    p->lists, p->select_counters, p->beam_keys, p->beam_sums, p->staging};
    for (void *b : bufs)
        if (b) (void)hipFree(b);
    if (p->stream) (void)hipStreamDestroy(p->stream);
    delete p;
    return 0;
}

const char *leap_hip_attention_pages_last_error(const leap_hip_attention_pages *p) { return p ? p->err.c_str() : g_pages_error; }

int leap_hip_attention_pages_clear(leap_hip_attention_pages *p)
{
    if (!p) return -EINVAL;
    HIP_TRY(p, hipSetDevice(p->cfg.model.device));
    return clear_all(p);
}

int leap_hip_attention_pages_state(leap_hip_attention_pages *p, int *table, int *refs)
{
    if (!p) return -EINVAL;
    HIP_TRY(p, hipSetDevice(p->cfg.model.device));
    const size_t entries = (size_t)p->cfg.model.max_batch * p->width;
    if (table) HIP_TRY(p, hipMemcpyAsync(table, p->table, entries * sizeof(int), hipMemcpyDeviceToHost, p->stream));
    if (refs) HIP_TRY(p, hipMemcpyAsync(refs, p->refs, (size_t)p->cfg.n_pages * sizeof(int), hipMemcpyDeviceToHost, p->stream));
    HIP_TRY(p, hipStreamSynchronize(p->stream));
    return 0;
}

int leap_hip_attention_pages_view(leap_hip_attention_pages *p, int layer, leap_hip_attention_pages_arrays *out)
{
    if (!p) return -EINVAL;
    if (int rc = check_layer(p, layer)) return rc;
    if (!out) return set_err(p, -EINVAL, "out is NULL");
    *out = {p->table, p->refs, p->width, layer_at<void>(p, 0, layer), layer_at<void>(p, 1, layer),
            p->q8 ? layer_at<float>(p, 2, layer) : nullptr, p->q8 ? layer_at<float>(p, 3, layer) : nullptr,
            p->cfg.bounds ? layer_at<float>(p, 4, layer) : nullptr};
    return 0;
}

// ---- tables ------------------------------------------------------------------------

int leap_hip_attention_pages_reserve_async(leap_hip_attention_pages *p, int n_seq, const int *begin, const int *end, int *status,
                                           void *stream)
{
    if (!p) return -EINVAL;
    if (int rc = check_seqs(p, n_seq)) return rc;
    if (!begin || !end) return set_err(p, -EINVAL, "NULL buffer");
    if (!aligned(begin, 4) || !aligned(end, 4) || !aligned(status, 4))
        return set_err(p, -EINVAL, "begin, end and status must be 4-byte aligned");
    HIP_TRY(p, hipSetDevice(p->cfg.model.device));
    return launch_reserve(p, n_seq, begin, end, status, (hipStream_t)stream);
}

int leap_hip_attention_pages_reserve(leap_hip_attention_pages *p, int n_seq, const int *begin, const int *end)
{
    if (!p) return -EINVAL;
    if (int rc = check_seqs(p, n_seq)) return rc;
    if (!begin || !end) return set_err(p, -EINVAL, "NULL buffer");
    for (int i = 0; i < n_seq; i++)
        if (begin[i] < 0 || begin[i] > end[i] || end[i] > p->cfg.model.seq_len)
            return set_err(p, -EINVAL, "sequence %d: rows [%d, %d) outside [0, %d)", i, begin[i], end[i], p->cfg.model.seq_len);
    int status = 0;
    // (-ENOMEM is the pool's alone: who gets it can free pages, or wait)
    if (int rc = reserve_host(p, n_seq, begin, end, &status)) return rc == -ENOMEM ? -EIO : rc;
    return status ? set_err(p, status, "the pool of %d pages has too few free ones", p->cfg.n_pages) : 0;
}

int leap_hip_attention_pages_fork_async(leap_hip_attention_pages *p, int n_seq, const int *parent, const int *rows, void *stream)
{
    if (!p) return -EINVAL;
    if (int rc = check_seqs(p, n_seq)) return rc;
    if (!rows) return set_err(p, -EINVAL, "NULL buffer");
    if (!aligned(parent, 4) || !aligned(rows, 4)) return set_err(p, -EINVAL, "parent and rows must be 4-byte aligned");
    HIP_TRY(p, hipSetDevice(p->cfg.model.device));
    return launch_fork(p, n_seq, parent, rows, (hipStream_t)stream);
}

int leap_hip_attention_pages_fork(leap_hip_attention_pages *p, int n_seq, const int *parent, const int *rows)
{
    if (!p) return -EINVAL;
    if (int rc = check_seqs(p, n_seq)) return rc;
    if (!rows) return set_err(p, -EINVAL, "NULL buffer");
    for (int i = 0; i < n_seq; i++) {
        if (parent && (parent[i] < 0 || parent[i] >= p->cfg.model.max_batch))
            return set_err(p, -EINVAL, "parent[%d] = %d outside [0, %d)", i, parent[i], p->cfg.model.max_batch);
        if (rows[i] < 0 || rows[i] > p->cfg.model.seq_len)
            return set_err(p, -EINVAL, "rows[%d] = %d outside [0, %d]", i, rows[i], p->cfg.model.seq_len);
    }
    HIP_TRY(p, hipSetDevice(p->cfg.model.device));
    const size_t bytes = (size_t)n_seq * sizeof(int);
    if (int rc = staging(p, 2 * bytes)) return rc;
    int *rd = reinterpret_cast<int *>(p->staging), *pd = rd + n_seq;
    HIP_TRY(p, hipMemcpyAsync(rd, rows, bytes, hipMemcpyHostToDevice, p->stream));
    if (parent) HIP_TRY(p, hipMemcpyAsync(pd, parent, bytes, hipMemcpyHostToDevice, p->stream));
    if (int rc = launch_fork(p, n_seq, parent ? pd : nullptr, rd, p->stream)) return rc;
    HIP_TRY(p, hipStreamSynchronize(p->stream));
    return 0;
}

int leap_hip_attention_pages_compact_async(leap_hip_attention_pages *p, int *used, void *stream)
{
    if (!p) return -EINVAL;
    if (!aligned(used, 4)) return set_err(p, -EINVAL, "used must be 4-byte aligned");
    HIP_TRY(p, hipSetDevice(p->cfg.model.device));
    leap::PagesArgs a = pages_args(p, p->cfg.model.max_batch);
    a.count = used;
    HIP_TRY(p, launch_k(leap::compact_kernel, dim3(1), dim3(leap::kPlanThreads), (hipStream_t)stream, a));
    return launch_copies(p, true, (hipStream_t)stream);
}

int leap_hip_attention_pages_compact(leap_hip_attention_pages *p, int *used)
{
    if (!p) return -EINVAL;
    HIP_TRY(p, hipSetDevice(p->cfg.model.device));
    if (int rc = staging(p, sizeof(int))) return rc;
    int *d = reinterpret_cast<int *>(p->staging), n = 0;
    if (int rc = leap_hip_attention_pages_compact_async(p, d, p->stream)) return rc;
    HIP_TRY(p, hipMemcpyAsync(&n, d, sizeof n, hipMemcpyDeviceToHost, p->stream));
    HIP_TRY(p, hipStreamSynchronize(p->stream));
    if (used) *used = n;
    return 0;
}

// ---- the step ------------------------------------------------------------------------

int leap_hip_attention_pages_step_async(leap_hip_attention_pages *p, int layer, int n_seq, const int *pos, int max_pos,
                                        long long total_rows, const float *q, const float *k_new, const float *v_new, float *out,
                                        void *stream)
{
    if (!p) return -EINVAL;
    if (int rc = step_checks(p, layer, n_seq, pos, max_pos, total_rows, q, k_new, v_new, out)) return rc;
    HIP_TRY(p, hipSetDevice(p->cfg.model.device));
    // (without a count, as if the sequences were spread evenly up to the longest)
    const long long rows = total_rows > 0 ? total_rows : n_seq == 1 ? max_pos + 1 : (long long)n_seq * (max_pos + 1) / 2 + 1;
    return launch_step(p, layer, n_seq, pos, max_pos, rows, 0, q, k_new, v_new, out, (hipStream_t)stream);
}

int leap_hip_attention_pages_step_sparse_async(leap_hip_attention_pages *p, int layer, int n_seq, const int *pos, int max_pos,
                                               int keep, const float *q, const float *k_new, const float *v_new, float *out,
                                               int *picked, void *stream)
{
    if (!p) return -EINVAL;
    if (!p->cfg.bounds) return set_err(p, -EINVAL, "the sparse step needs a handle with bounds");
    if (keep < 1) return set_err(p, -EINVAL, "keep %d is not positive", keep);
    if (int rc = step_checks(p, layer, n_seq, pos, max_pos, 0, q, k_new, v_new, out)) return rc;
    if (!aligned(picked, 4)) return set_err(p, -EINVAL, "picked must be 4-byte aligned");
    HIP_TRY(p, hipSetDevice(p->cfg.model.device));
    const int most = std::min(keep, p->width);
    if (int rc = launch_select(p, layer, n_seq, pos, max_pos, most, keep, q, picked, (hipStream_t)stream)) return rc;
    return launch_step(p, layer, n_seq, pos, max_pos, 0, most, q, k_new, v_new, out, (hipStream_t)stream);
}

static int step_host(leap_hip_attention_pages *p, int layer, int n_seq, const int *pos, int keep, const float *q, const float *k_new,
                     const float *v_new, float *out, int *picked)
{
    if (!p) return -EINVAL;
    if (int rc = check_layer(p, layer)) return rc;
    if (int rc = check_seqs(p, n_seq)) return rc;
    if (!pos || !q || !k_new || !v_new || !out) return set_err(p, -EINVAL, "NULL buffer");
    int max_pos = 0;
    long long rows = 0;
    for (int i = 0; i < n_seq; i++) {
        if (pos[i] < 0 || pos[i] >= p->cfg.model.seq_len)
            return set_err(p, -EINVAL, "pos[%d] = %d outside [0, %d)", i, pos[i], p->cfg.model.seq_len);
        max_pos = std::max(max_pos, pos[i]);
        rows += pos[i] + 1;
    }
    HIP_TRY(p, hipSetDevice(p->cfg.model.device));
    const size_t qn = (size_t)n_seq * p->q_dim, kn = (size_t)n_seq * p->kv_dim;
    const size_t pn = picked ? (size_t)n_seq * p->cfg.model.n_kv_heads * keep : 0;
    if (int rc = staging(p, (2 * qn + 2 * kn) * sizeof(float) + (n_seq + pn) * sizeof(int))) return rc;
    float *qd = reinterpret_cast<float *>(p->staging), *kd = qd + qn, *vd = kd + kn, *od = vd + kn;
    int *xd = reinterpret_cast<int *>(od + qn), *cd = xd + n_seq;
    hipStream_t s = p->stream;
    HIP_TRY(p, hipMemcpyAsync(qd, q, qn * sizeof(float), hipMemcpyHostToDevice, s));
    HIP_TRY(p, hipMemcpyAsync(kd, k_new, kn * sizeof(float), hipMemcpyHostToDevice, s));
    HIP_TRY(p, hipMemcpyAsync(vd, v_new, kn * sizeof(float), hipMemcpyHostToDevice, s));
    HIP_TRY(p, hipMemcpyAsync(xd, pos, n_seq * sizeof(int), hipMemcpyHostToDevice, s));
    const int rc = keep ? leap_hip_attention_pages_step_sparse_async(p, layer, n_seq, xd, max_pos, keep, qd, kd, vd, od, picked ? cd : nullptr, s)
                        : leap_hip_attention_pages_step_async(p, layer, n_seq, xd, max_pos, rows, qd, kd, vd, od, s);
    if (rc) return rc;
    HIP_TRY(p, hipMemcpyAsync(out, od, qn * sizeof(float), hipMemcpyDeviceToHost, s));
    if (picked) HIP_TRY(p, hipMemcpyAsync(picked, cd, pn * sizeof(int), hipMemcpyDeviceToHost, s));
    HIP_TRY(p, hipStreamSynchronize(s));
    return 0;
}

int leap_hip_attention_pages_step(leap_hip_attention_pages *p, int layer, int n_seq, const int *pos, const float *q,
                                  const float *k_new, const float *v_new, float *out)
{
    return step_host(p, layer, n_seq, pos, 0, q, k_new, v_new, out, nullptr);
}

int leap_hip_attention_pages_step_sparse(leap_hip_attention_pages *p, int layer, int n_seq, const int *pos, int keep, const float *q,
                                         const float *k_new, const float *v_new, float *out, int *picked)
{
    if (!p) return -EINVAL;
    if (!p->cfg.bounds) return set_err(p, -EINVAL, "the sparse step needs a handle with bounds");
    if (keep < 1) return set_err(p, -EINVAL, "keep %d is not positive", keep);
    return step_host(p, layer, n_seq, pos, keep, q, k_new, v_new, out, picked);
}

// ---- rows ------------------------------------------------------------------------------

int leap_hip_attention_pages_write_async(leap_hip_attention_pages *p, int seq, int layer, int pos_begin, int pos_end, const float *k,
                                         const float *v, void *stream)
{
    return rows_async(p, seq, layer, pos_begin, pos_end, k, v, nullptr, nullptr, stream);
}
int leap_hip_attention_pages_read_async(leap_hip_attention_pages *p, int seq, int layer, int pos_begin, int pos_end, float *k, float *v,
                                        void *stream)
{
    return rows_async(p, seq, layer, pos_begin, pos_end, nullptr, nullptr, k, v, stream);
}
int leap_hip_attention_pages_write(leap_hip_attention_pages *p, int seq, int layer, int pos_begin, int pos_end, const float *k,
                                   const float *v)
{
    return rows_host(p, seq, layer, pos_begin, pos_end, k, v, nullptr, nullptr);
}
int leap_hip_attention_pages_read(leap_hip_attention_pages *p, int seq, int layer, int pos_begin, int pos_end, float *k, float *v)
{
    return rows_host(p, seq, layer, pos_begin, pos_end, nullptr, nullptr, k, v);
}

// ---- beams -----------------------------------------------------------------------------

int leap_hip_attention_pages_beam_select_async(leap_hip_attention_pages *p, int n_groups, int beams, int vocab, const float *logits,
                                               long long stride, const float *score, int *parent, int *token, float *best,
                                               void *stream)
{
    if (!p) return -EINVAL;
    if (int rc = beam_checks(p, n_groups, beams, vocab, logits, stride, score, parent, token, best)) return rc;
    HIP_TRY(p, hipSetDevice(p->cfg.model.device));
    return launch_beam(p, n_groups, beams, vocab, logits, stride, score, parent, token, best, (hipStream_t)stream);
}

int leap_hip_attention_pages_beam_select(leap_hip_attention_pages *p, int n_groups, int beams, int vocab, const float *logits,
                                         const float *score, int *parent, int *token, float *best)
{
    if (!p) return -EINVAL;
    if (int rc = beam_checks(p, n_groups, beams, vocab, logits, vocab, score, parent, token, best)) return rc;
    HIP_TRY(p, hipSetDevice(p->cfg.model.device));
    const size_t rows = (size_t)n_groups * beams, n = rows * vocab;
    if (int rc = staging(p, (n + rows) * sizeof(float) + rows * (2 * sizeof(int) + sizeof(float)))) return rc;
    float *ld = reinterpret_cast<float *>(p->staging), *sd = ld + n, *bd = sd + rows;
    int *pd = reinterpret_cast<int *>(bd + rows), *td = pd + rows;
    hipStream_t s = p->stream;
    HIP_TRY(p, hipMemcpyAsync(ld, logits, n * sizeof(float), hipMemcpyHostToDevice, s));
    HIP_TRY(p, hipMemcpyAsync(sd, score, rows * sizeof(float), hipMemcpyHostToDevice, s));
    if (int rc = launch_beam(p, n_groups, beams, vocab, ld, vocab, sd, pd, td, bd, s)) return rc;
    HIP_TRY(p, hipMemcpyAsync(parent, pd, rows * sizeof(int), hipMemcpyDeviceToHost, s));
    HIP_TRY(p, hipMemcpyAsync(token, td, rows * sizeof(int), hipMemcpyDeviceToHost, s));
    HIP_TRY(p, hipMemcpyAsync(best, bd, rows * sizeof(float), hipMemcpyDeviceToHost, s));
    HIP_TRY(p, hipStreamSynchronize(s));
    return 0;
}

}  // extern "C"
