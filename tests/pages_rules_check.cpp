// Host-side check of caches of pages on the library's own source, without a
// device: HIP's calls are stood in for by functions on host memory, which can
// be told to fail.  Built and run by tests/test_pages_rules.py.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>

namespace stand_in {
bool no_memory = false;       // every allocation fails
bool no_copy_memory = false;  // every copy fails for want of memory
int allocations = 0;
int status = 0;  // what the device answers to a reservation

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
#define hipLaunchKernel(...) hipSuccess
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

}  // namespace

int main()
{
    check_out_of_memory();
    std::puts("ok");
}
