// hip_on_host.cpp — the HIP runtime's functions that the library's host code calls, on host memory: allocations are the heap's, copies are memcpy, launches are
// counted and do nothing.  Loaded with RTLD_GLOBAL in front of the library, so the library's own host code runs as it is, without a GPU.  Failures are the test's.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <map>

static thread_local hipError_t g_last = hipSuccess;          // a failed call's error, until somebody asks
static hipError_t done(hipError_t e) { if (e != hipSuccess) g_last = e; return e; }
static int g_fail_malloc = 0, g_fail_host_malloc = 0, g_fail_launch = 0;             // the n-th from now fails
static uint64_t g_launches = 0, g_most_threads = 0, g_blocks = 0;
static std::map<void*, size_t> g_held;

extern "C" {
#define FAKE __attribute__((visibility("default")))
FAKE void fake_fail_malloc(int n) { g_fail_malloc = n; }
FAKE void fake_fail_host_malloc(int n) { g_fail_host_malloc = n; }
FAKE void fake_fail_launch(int n) { g_fail_launch = n; }
FAKE void fake_reset() { g_launches = g_most_threads = g_blocks = 0; }
FAKE uint64_t fake_launches() { return g_launches; }
FAKE uint64_t fake_most_threads() { return g_most_threads; }          // of one launch
FAKE uint64_t fake_blocks() { return g_blocks; }                      // workgroups of all launches
FAKE int fake_pending() { return (int)g_last; }
FAKE int fake_holds(const void* bytes, size_t n) {                     // allocations that begin with these bytes
    int found = 0;
    for (const auto& a : g_held) found += a.second >= n && memcmp(a.first, bytes, n) == 0;
    return found;
}

FAKE hipError_t hipMalloc(void** p, size_t n) {
    if (g_fail_malloc && --g_fail_malloc == 0) return done(hipErrorOutOfMemory);
    *p = calloc(1, n ? n : 1);
    if (!*p) return done(hipErrorOutOfMemory);
    g_held[*p] = n;
    return hipSuccess;
}
FAKE hipError_t hipFree(void* p) { g_held.erase(p); free(p); return hipSuccess; }
FAKE hipError_t hipExtMallocWithFlags(void** p, size_t n, unsigned) { return hipMalloc(p, n); }
FAKE hipError_t hipHostMalloc(void** p, size_t n, unsigned) {
    if (g_fail_host_malloc && --g_fail_host_malloc == 0) return done(hipErrorOutOfMemory);
    *p = calloc(1, n ? n : 1);
    return *p ? hipSuccess : done(hipErrorOutOfMemory);
}
FAKE hipError_t hipHostFree(void* p) { free(p); return hipSuccess; }
FAKE hipError_t hipMemcpy(void* d, const void* s, size_t n, hipMemcpyKind) { memcpy(d, s, n); return hipSuccess; }
FAKE hipError_t hipMemcpyAsync(void* d, const void* s, size_t n, hipMemcpyKind, hipStream_t) { memcpy(d, s, n); return hipSuccess; }
FAKE hipError_t hipMemcpy2D(void* d, size_t dp, const void* s, size_t sp, size_t w, size_t h, hipMemcpyKind) {
    for (size_t i = 0; i < h; ++i) memcpy((char*)d + i * dp, (const char*)s + i * sp, w);
    return hipSuccess;
}
FAKE hipError_t hipMemset(void* d, int v, size_t n) { memset(d, v, n); return hipSuccess; }
FAKE hipError_t hipMemsetAsync(void* d, int v, size_t n, hipStream_t) { memset(d, v, n); return hipSuccess; }
FAKE hipError_t hipSetDevice(int d) { return d == 0 ? hipSuccess : done(hipErrorInvalidDevice); }
FAKE hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
FAKE hipError_t hipGetDeviceCount(int* n) { *n = 1; return hipSuccess; }
FAKE hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int) {
    memset(p, 0, sizeof(*p));
    strcpy(p->gcnArchName, "gfx950");
    p->multiProcessorCount = 256;
    return hipSuccess;
}
FAKE hipError_t hipDeviceSynchronize() { return hipSuccess; }
FAKE hipError_t hipStreamCreate(hipStream_t* s) { *s = nullptr; return hipSuccess; }
FAKE hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) { *s = nullptr; return hipSuccess; }
FAKE hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
FAKE hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
FAKE hipError_t hipStreamGetDevice(hipStream_t, int* d) { *d = 0; return hipSuccess; }
FAKE hipError_t hipEventCreate(hipEvent_t* e) { *e = nullptr; return hipSuccess; }
FAKE hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) { *e = nullptr; return hipSuccess; }
FAKE hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
FAKE hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
FAKE hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
FAKE hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return hipSuccess; }
FAKE hipError_t hipGetLastError() { const hipError_t e = g_last; g_last = hipSuccess; return e; }
FAKE hipError_t hipLaunchKernel(const void*, dim3 g, dim3 b, void**, size_t, hipStream_t) {
    const uint64_t blocks = (uint64_t)g.x * g.y * g.z, threads = (uint64_t)b.x * b.y * b.z;
    ++g_launches;
    g_blocks += blocks;
    g_most_threads = blocks * threads > g_most_threads ? blocks * threads : g_most_threads;
    if (g_fail_launch && --g_fail_launch == 0) return done(hipErrorLaunchFailure);
    for (const uint64_t n : {(uint64_t)g.x * b.x, (uint64_t)g.y * b.y, (uint64_t)g.z * b.z})
        if (n == 0 || n >> 32) return done(hipErrorInvalidConfiguration);          // as the runtime does
    return hipSuccess;
}
}
