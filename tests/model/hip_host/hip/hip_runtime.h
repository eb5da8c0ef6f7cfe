// Host stand-in for the few runtime calls of np_devalloc.h (test infrastructure only): memory from malloc, streams and events as objects that
// remember whether they were destroyed.  A call on a destroyed stream is counted, and one that a stream is destroyed under is as well.
#pragma once
#include <atomic>
#include <chrono>
#include <cstdlib>
#include <cstring>
#include <thread>

enum hipError_t { hipSuccess = 0, hipErrorOutOfMemory = 2, hipErrorNotReady = 600 };
struct fake_stream { std::atomic<bool> gone{false}, busy{false}; };
struct fake_event { std::atomic<bool> done{true}; fake_stream* on = nullptr; };
typedef fake_stream* hipStream_t;
typedef fake_event* hipEvent_t;
constexpr unsigned hipStreamNonBlocking = 1, hipEventDisableTiming = 2, hipHostMallocPortable = 1;

struct fake_hip {
    std::atomic<int> used_destroyed{0}, mallocs{0}, frees{0}, host_mallocs{0}, host_frees{0}, in_call{0}, slow_ms{0};
    std::atomic<size_t> room{(size_t)-1};      // bytes hipMalloc still has
};
inline fake_hip& fake() { static fake_hip f; return f; }

// a call that takes slow_ms and uses the stream until its end
inline void fake_use(hipStream_t q) {
    if (!q) return;
    fake_hip& f = fake();
    if (q->gone) ++f.used_destroyed;
    ++f.in_call;
    if (f.slow_ms) std::this_thread::sleep_for(std::chrono::milliseconds(f.slow_ms.load()));
    --f.in_call;
    if (q->gone) ++f.used_destroyed;
}
inline hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
inline hipError_t hipGetLastError() { return hipSuccess; }
inline const char* hipGetErrorString(hipError_t) { return "error"; }
inline hipError_t hipMalloc(void** p, size_t n) {
    if (n > fake().room) { *p = nullptr; return hipErrorOutOfMemory; }
    ++fake().mallocs;
    *p = malloc(n);
    return hipSuccess;
}
inline hipError_t hipFree(void* p) { ++fake().frees; free(p); return hipSuccess; }
inline hipError_t hipHostMalloc(void** p, size_t n, unsigned) { ++fake().host_mallocs; *p = malloc(n); return hipSuccess; }
inline hipError_t hipHostFree(void* p) { ++fake().host_frees; free(p); return hipSuccess; }
inline hipError_t hipMemsetAsync(void* p, int v, size_t n, hipStream_t q) { fake_use(q); memset(p, v, n); return hipSuccess; }
inline hipError_t hipStreamCreateWithFlags(hipStream_t* q, unsigned) { *q = new fake_stream(); return hipSuccess; }
inline hipError_t hipStreamDestroy(hipStream_t q) { q->gone = true; return hipSuccess; }      // (the object itself stays: late uses are counted)
inline hipError_t hipStreamQuery(hipStream_t q) { fake_use(q); return q && q->busy ? hipErrorNotReady : hipSuccess; }
inline hipError_t hipStreamSynchronize(hipStream_t q) { fake_use(q); if (q) q->busy = false; return hipSuccess; }
inline hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) { *e = new fake_event(); return hipSuccess; }
inline hipError_t hipEventRecord(hipEvent_t e, hipStream_t q) { fake_use(q); e->on = q; return hipSuccess; }
inline hipError_t hipEventQuery(hipEvent_t e) { return e->on && e->on->busy ? hipErrorNotReady : hipSuccess; }
inline hipError_t hipEventSynchronize(hipEvent_t e) { if (e->on) e->on->busy = false; return hipSuccess; }
