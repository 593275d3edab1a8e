// Host-side check of caches of pages on the library's own source, without a
// device: HIP's calls are stood in for by functions on host memory, which can
// be told to fail and which note what is launched.  "memory": what a failed
// allocation or copy does.  "launches": over head shapes, both types, batches
// and lengths, a step's runs cover every tile once, each with records of its
// own inside the workspace and a group's within a merge's reach, and a choice's
// workgroups cover every page and count inside their counters.  Built and run
// by tests/test_pages_rules.py.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <set>
#include <vector>

namespace stand_in {
bool no_memory = false;       // every allocation fails
bool no_copy_memory = false;  // every copy fails for want of memory
int allocations = 0;
int status = 0;  // what the device answers to a reservation
struct Launch {
    const void *kernel;
    unsigned workgroups;
    std::vector<char> args;  // (of the first argument)
};
std::vector<Launch> launches;
bool noting = false;
size_t args_bytes[3];  // how much of it is noted, of each launch

hipError_t alloc(void **p, size_t n)
{
    if (no_memory) return hipErrorOutOfMemory;
    allocations++;
    return (*p = std::calloc(n ? n : 1, 1)) ? hipSuccess : hipErrorOutOfMemory;
}
hipError_t copy(void *to, const void *from, size_t n, hipMemcpyKind kind, hipStream_t)
{
    if (no_copy_memory) return hipErrorOutOfMemory;
    if (kind == hipMemcpyDeviceToHost && n == sizeof status)
        std::memcpy(to, &status, n);
    else
        std::memcpy(to, from, n);
    return hipSuccess;
}
hipError_t launch(const void *kernel, dim3 grid, dim3, void **args, size_t, hipStream_t)
{
    const char *a = static_cast<const char *>(args[0]);
    if (noting && launches.size() < 3) launches.push_back({kernel, grid.x * grid.y * grid.z, {a, a + args_bytes[launches.size()]}});
    return hipSuccess;
}
hipError_t attribute(int *out)
{
    *out = 256;
    return hipSuccess;
}
}  // namespace stand_in

#define hipMalloc(p, n) stand_in::alloc((void **)(p), n)
#define hipFree(p) (std::free(p), hipSuccess)
#define hipMemcpyAsync stand_in::copy
#define hipMemsetAsync(p, x, n, s) (std::memset(p, x, n), hipSuccess)
#define hipStreamSynchronize(s) hipSuccess
#define hipStreamCreate(s) hipSuccess
#define hipSetDevice(d) hipSuccess
#define hipGetDeviceCount(n) (*(n) = 1, hipSuccess)
#define hipDeviceGetAttribute(p, a, d) stand_in::attribute(p)
#define hipFuncGetAttributes(a, f) hipSuccess
#define hipLaunchKernel stand_in::launch
#define hipGetLastError() hipSuccess

#include "leap_hip_pages.hip"

int leap_host::check_placement(int, int, std::string *) { return 0; }

#define REQUIRE(c)                                                                                                     \
    do {                                                                                                               \
        if (!(c)) {                                                                                                    \
            std::printf("line %d: %s\n", __LINE__, #c);                                                                \
            std::exit(1);                                                                                              \
        }                                                                                                              \
    } while (0)

namespace {

leap_hip_attention_pages *handle(int n_heads, int n_kv, int hd, int seq_len, int max_batch, int page_rows, int n_pages, int q8, int bounds)
{
    leap_hip_attention_pages_config c{};
    c.model = {1, 0, 1, n_heads, n_kv, hd, seq_len, 0.0f, max_batch, 0};
    c.page_rows = page_rows;
    c.n_pages = n_pages;
    c.q8 = q8;
    c.bounds = bounds;
    leap_hip_attention_pages *p = nullptr;
    REQUIRE(leap_hip_attention_pages_create(&c, &p) == 0);
    return p;
}

// Tables change without memory being asked for (the pool may hold all there
// is), and only a pool with too few free pages is -ENOMEM.
void check_out_of_memory()
{
    constexpr int n = 300;
    leap_hip_attention_pages *p = handle(8, 2, 64, 64, n, 16, 4, 0, 0);
    int zero[n] = {}, one[n], used = 0;
    for (int &x : one) x = 1;
    const int before = stand_in::allocations;
    stand_in::no_memory = true;
    REQUIRE(leap_hip_attention_pages_reserve(p, n, zero, one) == 0);
    REQUIRE(leap_hip_attention_pages_fork(p, n, zero, one) == 0);
    REQUIRE(leap_hip_attention_pages_compact(p, &used) == 0);
    REQUIRE(stand_in::allocations == before);
    stand_in::status = -ENOMEM;
    REQUIRE(leap_hip_attention_pages_reserve(p, n, zero, one) == -ENOMEM);
    REQUIRE(std::strstr(leap_hip_attention_pages_last_error(p), "too few free"));
    stand_in::no_copy_memory = true;
    REQUIRE(leap_hip_attention_pages_reserve(p, n, zero, one) == -EIO);
    REQUIRE(std::strstr(leap_hip_attention_pages_last_error(p), "hipMemcpyAsync"));
    stand_in::no_memory = stand_in::no_copy_memory = false;
    stand_in::status = 0;
    leap_hip_attention_pages_destroy(p);
}

// From here on the launches are noted: the first has `first` bytes of arguments, the others are steps'.
void note(size_t first)
{
    stand_in::launches.clear();
    stand_in::args_bytes[0] = first;
    stand_in::args_bytes[1] = stand_in::args_bytes[2] = sizeof(leap::PagedArgs);
    stand_in::noting = true;
}

int n_flat = 0, n_spread = 0, n_split = 0, n_whole = 0;

// A step's launch (the last but one where its records are added up by another).
void check_step(leap_hip_attention_pages *p, const std::vector<int> &rows, int keep, bool told)
{
    const auto &m = p->cfg.model;
    const int n_seq = (int)rows.size(), tk = leap::paged_tile(m.head_dim, p->q8), R = p->cfg.page_rows;
    const int longest = *std::max_element(rows.begin(), rows.end());
    long long total = 0;
    for (int r : rows) total += r;
    alignas(16) static char buffer[64];  // (nothing reads it)
    int *pos = reinterpret_cast<int *>(buffer);
    float *x = reinterpret_cast<float *>(buffer);
    note(keep ? sizeof(leap::SelectArgs) : sizeof(leap::PagedArgs));
    if (keep)
        REQUIRE(leap_hip_attention_pages_step_sparse_async(p, 0, n_seq, pos, longest - 1, keep, x, x, x, x, nullptr, nullptr) == 0);
    else
        REQUIRE(leap_hip_attention_pages_step_async(p, 0, n_seq, pos, longest - 1, told ? total : 0, x, x, x, x, nullptr) == 0);
    stand_in::noting = false;
    const size_t at = keep ? 1 : 0;
    REQUIRE(stand_in::launches.size() > at);
    const stand_in::Launch &l = stand_in::launches[at];
    leap::PagedArgs a;
    std::memcpy(&a, l.args.data(), sizeof a);
    const PagedKernels fn = pick_paged(m.head_dim, p->group, p->q8);
    const int groups = n_seq * m.n_kv_heads;
    // rows that a group attends to
    auto seen = [&](int gi) {
        const int r = rows[gi / m.n_kv_heads], pages = (r - 1) / R + 1;
        return keep && keep < pages ? (keep - 1) * R + (r - 1) % R + 1 : r;
    };
    auto tiles_of = [&](int gi) { return (seen(gi) + tk - 1) / tk; };
    if (l.kernel == reinterpret_cast<const void *>(fn.flat)) {
        REQUIRE(!keep && stand_in::launches.size() == 1 && l.workgroups % leap::kXcds == 0);
        n_flat++;
        const int n_wg = (int)l.workgroups / leap::kXcds;
        REQUIRE(n_wg <= leap::kPagedSplits && (size_t)groups <= kCounters && !a.spread);
        std::set<size_t> records;
        for (int xcd = 0; xcd < leap::kXcds; xcd++) {
            const int items = (groups - xcd + leap::kXcds - 1) / leap::kXcds;
            REQUIRE(items >= 1 && items <= leap::kWave && items <= a.splits);
            std::vector<int> len(items), end(items), done(items, 0), runs(items, 0), n(items, 0);
            int sum = 0;
            for (int i = 0; i < items; i++) end[i] = sum += len[i] = tiles_of(i * leap::kXcds + xcd) + leap::kPagedStart;
            const int length = leap::paged_length(sum, n_wg);
            for (int w = 0; w < n_wg; w++) {
                const int stop = std::min((w + 1) * length, sum);
                for (int from = w * length; from < stop;) {
                    int i = 0;
                    while (end[i] <= from) i++;
                    const leap::PagedSegment g = leap::paged_segment(w, length, from, stop, i, len[i], end[i]);
                    from = end[i];
                    if (g.t1 <= g.t0) continue;
                    REQUIRE(g.t0 == done[i] && g.run == runs[i] && (runs[i] == 0 || g.n == n[i]));
                    done[i] = g.t1;
                    runs[i]++;
                    n[i] = g.n;
                    const size_t record = (size_t)xcd * (n_wg + a.splits) + g.record + g.run;
                    REQUIRE(g.n == 1 || records.insert(record).second);
                    REQUIRE((record + 1) * p->group <= kRecords);
                }
            }
            for (int i = 0; i < items; i++) REQUIRE(done[i] + leap::kPagedStart == len[i] && runs[i] == n[i] && n[i] <= leap::kPagedSplits);
        }
        return;
    }
    REQUIRE(l.kernel == reinterpret_cast<const void *>(fn.attention));
    (a.spread ? n_spread : a.splits > 1 ? n_split : n_whole)++;
    REQUIRE(a.chunk >= 1 && a.splits >= 1 && a.splits <= leap::kPagedSplits);
    const long long items = (groups + leap::kXcds - 1) / leap::kXcds;
    REQUIRE((long long)l.workgroups == (a.spread ? (long long)groups * a.splits : items * leap::kXcds * a.splits));
    if (a.splits > 1) REQUIRE((size_t)groups * a.splits * p->group <= kRecords && (size_t)groups <= kCounters);
    REQUIRE((stand_in::launches.size() == at + 2) == (a.spread != 0));
    if (a.spread) REQUIRE(stand_in::launches[at + 1].kernel == reinterpret_cast<const void *>(fn.merge) && (int)stand_in::launches[at + 1].workgroups == groups);
    for (int gi = 0; gi < groups; gi++) {
        REQUIRE((long long)a.chunk * a.splits >= tiles_of(gi));
        REQUIRE((int)leap::fast_div((uint32_t)(tiles_of(gi) + a.chunk - 1), a.by_chunk) == (tiles_of(gi) + a.chunk - 1) / a.chunk);
        REQUIRE(a.blocks * 16 >= seen(gi));
    }
    REQUIRE((a.blocks - 1) / (R / 16) < (keep ? std::max(a.keep, 1) : p->width));
}

void check_select(leap_hip_attention_pages *p, int n_seq, int longest, int keep)
{
    const auto &m = p->cfg.model;
    alignas(16) static char buffer[64];
    int *pos = reinterpret_cast<int *>(buffer);
    float *x = reinterpret_cast<float *>(buffer);
    note(sizeof(leap::SelectArgs));
    REQUIRE(leap_hip_attention_pages_step_sparse_async(p, 0, n_seq, pos, longest - 1, keep, x, x, x, x, nullptr, nullptr) == 0);
    stand_in::noting = false;
    const stand_in::Launch &l = stand_in::launches.at(0);
    REQUIRE(l.kernel == reinterpret_cast<const void *>(pick_paged(m.head_dim, p->group, p->q8).select));
    leap::SelectArgs a;
    std::memcpy(&a, l.args.data(), sizeof a);
    const int groups = n_seq * m.n_kv_heads;
    REQUIRE(a.units >= 1 && a.parts == (a.units + leap::kSelectPart - 1) / leap::kSelectPart && a.keep <= p->width);
    REQUIRE((long long)l.workgroups == (long long)(groups + leap::kXcds - 1) / leap::kXcds * leap::kXcds * a.units);
    const size_t counters = select_counters(p), first = (size_t)(a.part_counters - a.counters);
    REQUIRE(first >= (size_t)groups);
    if (a.units > 1) REQUIRE(first + ((size_t)groups * a.parts - 1) * leap::kCtrStride + 1 <= counters);
}

void check_launches()
{
    const int shapes[][3] = {{32, 8, 128}, {32, 4, 64}, {32, 32, 128}, {64, 8, 128}, {4, 1, 128}, {6, 3, 64}, {32, 2, 128}, {128, 8, 64}};
    unsigned long long seed = 1;
    auto pick = [&](int lo, int hi) {
        seed = seed * 6364136223846793005ull + 1442695040888963407ull;
        return lo + (int)((seed >> 33) % (unsigned long long)(hi - lo + 1));
    };
    for (const auto &s : shapes)
        for (int q8 = 0; q8 < 2; q8++) {
            leap_hip_attention_pages *p = handle(s[0], s[1], s[2], 131072, 600, 128, 4, q8, 1);
            for (int n_seq : {1, 2, 3, 7, 8, 9, 15, 16, 17, 20, 33, 40, 45, 64, 65, 130, 600})
                for (int longest : {1, 16, 17, 64, 65, 500, 2048, 4096, 8192, 70000, 131072})
                    for (int kind = 0; kind < 4; kind++) {
                        std::vector<int> rows(n_seq, longest);
                        for (int i = 1; i < n_seq && kind; i++) rows[i] = kind == 1 ? 1 : kind == 2 ? pick(1, longest) : pick((longest + 1) / 2, longest);
                        for (bool told : {false, true}) check_step(p, rows, 0, told);
                        if (kind != 1)
                            for (int keep : {1, 4, 64, 1024}) check_step(p, rows, keep, false);
                    }
            leap_hip_attention_pages_destroy(p);
            p = handle(s[0], s[1], s[2], 131072, 300, 16, 4, q8, 1);
            for (int n_seq : {1, 2, 3, 8, 9, 31, 32, 33, 64, 65, 128, 300})
                for (int longest : {1, 16, 17, 1000, 1025, 4096, 30000, 131072})
                    for (int keep : {1, 2, 100, 8192}) check_select(p, n_seq, longest, keep);
            leap_hip_attention_pages_destroy(p);
        }
    std::printf("%d flat launches, %d spread, %d split, %d whole\n", n_flat, n_spread, n_split, n_whole);
    REQUIRE(n_flat > 100 && n_spread > 100 && n_split > 100 && n_whole > 100);
}

}  // namespace

int main(int argc, char **argv)
{
    const char *what = argc > 1 ? argv[1] : "";
    if (!std::strcmp(what, "memory"))
        check_out_of_memory();
    else if (!std::strcmp(what, "launches"))
        check_launches();
    else
        return 2;
    std::puts("ok");
}
