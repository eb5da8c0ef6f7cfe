// Device allocations of both libraries go through here.
//
// A caching allocator in front of hipMalloc / hipFree (BlockCache below).  Why: on this runtime hipFree waits for work of OTHER streams
// (measured: a buffer that a 300 ms kernel of another non-blocking stream was writing took 300.3 ms to free, profiles/r5_fault_hunt.txt
// section 3), and a drop-in call or a tile allocates and frees ~110 buffers -- a long-lived worker (the reference's caller: one process,
// contig after contig, source/lib/nextpolish1.py:181-189,219-224) made ~65 000 such waits per run of the test suite, and the one-process
// suite was seen to stop inside a release.  With the cache a released buffer goes to a per-device free list and the
// next request of a similar size takes it from there: no runtime call on either side in steady state.  The guarantee hipFree gave --
// nothing in flight still touches the block when somebody else gets it -- is kept without waiting: at release time every stream either
// library created (stream_create below keeps the registry) is asked with hipStreamQuery; for each one that is busy an event is
// recorded and kept with the block, and the block is handed out again only once those events have completed (asked with
// hipEventQuery at the time of the request; a block that is not ready is skipped, the request falls through to hipMalloc).
// NP_DEVCACHE_MB=<n> bounds the idle bytes kept per device (default 16384, at least 256: with nothing kept, every release of the ~110 buffers
// of a call would be one to the runtime, the pattern in which a process was seen to stop); NP_PINCACHE_MB=<n> the same for page-locked host
// memory (default 2048).  Over the bound the largest idle blocks go back to the runtime, and when hipMalloc runs out of memory the cache is
// emptied and the request retried.
// Whenever memory does go back to the runtime, every stream is synchronised with hipStreamSynchronize first (quiesce below, and why).
//
// NP_DEVPOISON=1 (debugging; or a hex byte, e.g. NP_DEVPOISON=ff): every new device buffer is filled with that byte (default a5) before it
// is handed out.  hipMalloc hands a long-lived process the bytes of whatever it freed before -- a fresh process mostly sees zeros -- so a
// kernel that reads memory nobody wrote behaves differently in the one-process test suite than in any single test; with the poison it
// misbehaves the same way everywhere.  NP_DEVPOISON=2 also fills the work buffers of a short-read batch before
// every run (what an earlier run left in a reused buffer is the other thing only a long-lived process has).
#pragma once
#include <hip/hip_runtime.h>

#include <fcntl.h>
#include <sys/syscall.h>
#include <time.h>
#include <unistd.h>

#include <chrono>
#include <cstdio>
#include <cstdlib>
#include <cstdint>
#include <cstring>
#include <map>
#include <mutex>
#include <shared_mutex>
#include <unordered_map>
#include <vector>

namespace npalloc {

// NP_ALLOCLOG=<path> (debugging): every device allocation and pinned host allocation of both libraries, and every
// release, is appended to <path>.<pid> as one line "<ms> <tid> <op> <address> <bytes>" (ops D+ D- device, H+ H- hipHostMalloc),
// written with one write(2) each so that the file is complete when the runtime ends the process on a GPU memory fault:
// the address in the runtime's "Memory access fault by GPU ... on address" line is then looked up among the ranges that were live, or had
// just been released, at that moment (tests/tools/r5_fault_lookup.py).
inline int alloc_log_fd() {
    static const int fd = [] {
        const char* e = getenv("NP_ALLOCLOG");
        if (!e || !e[0]) return -1;
        char path[600];
        snprintf(path, sizeof path, "%.500s.%d", e, (int)getpid());
        return open(path, O_WRONLY | O_CREAT | O_APPEND, 0644);
    }();
    return fd;
}
inline void alloc_log(const char* op, const void* p, size_t bytes) {
    const int fd = alloc_log_fd();
    if (fd < 0) return;
    timespec ts;
    clock_gettime(CLOCK_MONOTONIC, &ts);
    char line[160];
    const int n = snprintf(line, sizeof line, "%lld.%03ld %ld %s %p %zu\n", (long long)ts.tv_sec, ts.tv_nsec / 1000000, (long)syscall(SYS_gettid), op, p, bytes);
    if (n > 0) (void)!write(fd, line, (size_t)n);
}

// Page-locked host memory of both libraries comes from here: hipHostMalloc, and a list of the ranges handed out -- np_hostcopy.h lets
// the DMA engines touch host memory only when it lies in one of them (never the user's pageable pages, never heap memory
// registered with the runtime).
struct PinnedRanges {
    std::mutex mu;
    std::map<uintptr_t, size_t> live;      // start -> bytes
};
inline PinnedRanges& pinned_ranges() { static PinnedRanges* r = new PinnedRanges(); return *r; }
inline bool is_pinned(const void* p, size_t bytes) {
    PinnedRanges& R = pinned_ranges();
    const uintptr_t a = (uintptr_t)p;
    std::lock_guard<std::mutex> g(R.mu);
    auto it = R.live.upper_bound(a);
    if (it == R.live.begin()) return false;
    --it;
    return a >= it->first && a + bytes <= it->first + it->second;
}
// (pinned host memory goes through a BlockCache of its own, defined below -- hipHostFree waits for the device like hipFree does)
inline hipError_t host_malloc(void** p, size_t bytes, unsigned flags);
inline hipError_t host_free(void* p);

// ----------------------------------------------------------------------------------------------- stream registry
// Streams of both libraries are created and destroyed through here, so that a released block can be fenced against everything in flight
// (BlockCache) and a stopped process can say which stream is busy (report below, used by the tests' watchdog).
// Whoever asks, waits for or records on streams of the registry holds `mu` shared until it is done with them; stream_destroy takes it alone
// to strike the stream off.  So a stream is never destroyed under a thread that releases memory at the same time.
struct StreamRegistry {
    std::shared_timed_mutex mu;
    std::map<hipStream_t, int> live;      // stream -> device
};
inline StreamRegistry& stream_registry() { static StreamRegistry* r = new StreamRegistry(); return *r; }
inline hipError_t stream_create(hipStream_t* q) {
    const hipError_t e = hipStreamCreateWithFlags(q, hipStreamNonBlocking);
    if (e == hipSuccess) {
        int dev = 0;
        (void)hipGetDevice(&dev);
        StreamRegistry& R = stream_registry();
        std::lock_guard<std::shared_timed_mutex> g(R.mu);
        R.live[*q] = dev;
    }
    return e;
}
// (hooks run before a stream goes away: the pinned copy ring settles the events it recorded on it, np_hostcopy.h)
typedef void (*StreamDestroyHook)(hipStream_t);
inline StreamDestroyHook& stream_destroy_hook() { static StreamDestroyHook h = nullptr; return h; }
inline hipError_t stream_destroy(hipStream_t q) {
    if (!q) return hipSuccess;
    (void)hipStreamSynchronize(q);
    if (StreamDestroyHook h = stream_destroy_hook()) h(q);
    {
        StreamRegistry& R = stream_registry();
        std::lock_guard<std::shared_timed_mutex> g(R.mu);
        R.live.erase(q);
    }
    return hipStreamDestroy(q);
}
// f(q) for every stream of `dev` (and the null stream) that still has work in flight
template <class F> inline void for_busy_streams(int dev, F f) {
    StreamRegistry& R = stream_registry();
    std::shared_lock<std::shared_timed_mutex> g(R.mu);
    for (auto& kv : R.live) if (kv.second == dev && hipStreamQuery(kv.first) == hipErrorNotReady) f(kv.first);
    if (hipStreamQuery(nullptr) == hipErrorNotReady) f((hipStream_t) nullptr);
}

// Before memory really goes back to the runtime.  hipFree and hipHostFree wait for work in flight on every stream, and a release was seen
// not to return at all: three stops of the test process inside this project's own release path (DevBuf::ensure, np1_batch_free; the last
// one in BlockCache::put with nothing kept, where it made one call, hipFree), while hipStreamQuery answered "ready" for every stream
// of the process (profiles/r6_hang_hunt.txt).  hipStreamSynchronize was not seen to stop.  So every stream of the registry and the null
// stream are synchronised with it first, under one lock so that two releasing threads do not interleave: the release itself then has no
// work in flight to wait for.
inline std::mutex& raw_free_mutex() { static std::mutex* m = new std::mutex(); return *m; }
inline void quiesce() {
    StreamRegistry& R = stream_registry();
    std::shared_lock<std::shared_timed_mutex> g(R.mu);
    for (auto& kv : R.live) (void)hipStreamSynchronize(kv.first);
    (void)hipStreamSynchronize(nullptr);
}

// ----------------------------------------------------------------------------------------------- block cache
struct CacheStats { uint64_t hits = 0, misses = 0, raw_frees = 0, fenced = 0, not_ready = 0, flushes = 0; size_t cached = 0, live = 0, peak_cached = 0; };

class BlockCache {
public:
    typedef hipError_t (*RawAlloc)(void**, size_t);
    typedef hipError_t (*RawFree)(void*);
    BlockCache(RawAlloc a, RawFree f, size_t cap_bytes) : alloc_(a), free_(f), cap_(cap_bytes) {}

    // size classes with three mantissa bits (at most 12.5 % above the request), 4 KiB at least
    static size_t size_class(size_t bytes) {
        if (bytes <= 4096) return 4096;
        int top = 63 - __builtin_clzll((unsigned long long)bytes);
        const size_t step = (size_t)1 << (top - 3);
        return (bytes + step - 1) & ~(step - 1);
    }

    hipError_t get(void** p, size_t bytes) {
        int dev = 0;
        (void)hipGetDevice(&dev);
        const size_t want = size_class(bytes);
        Block hit{};
        bool found = false;
        {
            std::lock_guard<std::mutex> g(mu_);
            auto& fl = free_list_[dev];
            // a block of up to 1.5x the class (small ones: up to 4x, nothing is lost with them)
            const size_t most = want < ((size_t)1 << 20) ? want * 4 : want + want / 2;
            int looked = 0;
            for (auto it = fl.lower_bound(want); it != fl.end() && it->first <= most && looked < 8; ++it, ++looked) {
                bool ready = true;
                for (hipEvent_t e : it->second.waits) if (hipEventQuery(e) != hipSuccess) { ready = false; break; }
                if (!ready) { ++st_.not_ready; continue; }
                hit = it->second;
                fl.erase(it);
                found = true;
                break;
            }
            if (found) {
                st_.cached -= hit.bytes;
                st_.live += hit.bytes;
                ++st_.hits;
                live_[hit.p] = Live{hit.bytes, dev};
                for (hipEvent_t e : hit.waits) spare_events_.push_back(e);
            }
        }
        if (found) { *p = hit.p; return hipSuccess; }
        hipError_t e = alloc_(p, want);
        if (e != hipSuccess) {
            (void)hipGetLastError();
            flush(dev);                      // out of memory with blocks of our own lying idle: give them back and ask again
            e = alloc_(p, want);
        }
        if (e == hipSuccess) {
            std::lock_guard<std::mutex> g(mu_);
            ++st_.misses;
            st_.live += want;
            live_[*p] = Live{want, dev};
        }
        return e;
    }

    hipError_t put(void* p) {
        if (!p) return hipSuccess;
        Live l{};
        {
            std::lock_guard<std::mutex> g(mu_);
            auto it = live_.find(p);
            if (it == live_.end()) { ++st_.raw_frees; l.bytes = 0; }
            else { l = it->second; live_.erase(it); st_.live -= l.bytes; }
        }
        if (l.bytes == 0 || l.bytes > cap_) {
            if (l.bytes) { std::lock_guard<std::mutex> g(mu_); ++st_.raw_frees; }
            std::lock_guard<std::mutex> g(raw_free_mutex());
            quiesce();
            return free_(p);
        }
        // fence the block against whatever is in flight on any stream of ours (what hipFree did by waiting)
        Block b{p, l.bytes, {}};
        for_busy_streams(l.dev, [&](hipStream_t q) {
            hipEvent_t e = take_event();
            if (!e || hipEventRecord(e, q) != hipSuccess) {      // cannot fence: wait like hipFree would have
                if (e) give_event(e);
                (void)hipStreamSynchronize(q);
                return;
            }
            b.waits.push_back(e);
        });
        std::vector<Block> evict;
        {
            std::lock_guard<std::mutex> g(mu_);
            if (!b.waits.empty()) ++st_.fenced;
            free_list_[l.dev].emplace(b.bytes, b);
            st_.cached += b.bytes;
            if (st_.cached > st_.peak_cached) st_.peak_cached = st_.cached;
            // over the bound: the largest idle blocks of this device go back to the runtime
            auto& fl = free_list_[l.dev];
            while (st_.cached > cap_ && !fl.empty()) {
                auto last = std::prev(fl.end());
                evict.push_back(last->second);
                st_.cached -= last->second.bytes;
                fl.erase(last);
            }
        }
        for (Block& v : evict) release_block(v);
        return hipSuccess;
    }

    // every idle block of the device back to the runtime (dev < 0: of every device)
    void flush(int dev) {
        std::vector<Block> all;
        {
            std::lock_guard<std::mutex> g(mu_);
            ++st_.flushes;
            for (auto& kv : free_list_) {
                if (dev >= 0 && kv.first != dev) continue;
                for (auto& b : kv.second) { all.push_back(b.second); st_.cached -= b.second.bytes; }
                kv.second.clear();
            }
        }
        for (Block& v : all) release_block(v);
    }
    CacheStats stats() { std::lock_guard<std::mutex> g(mu_); return st_; }
    size_t cap() const { return cap_; }

private:
    struct Block { void* p; size_t bytes; std::vector<hipEvent_t> waits; };
    struct Live { size_t bytes; int dev; };
    void release_block(Block& v) {
        for (hipEvent_t e : v.waits) { (void)hipEventSynchronize(e); give_event(e); }
        { std::lock_guard<std::mutex> g(mu_); ++st_.raw_frees; }
        std::lock_guard<std::mutex> g(raw_free_mutex());
        quiesce();
        (void)free_(v.p);
    }
    hipEvent_t take_event() {
        {
            std::lock_guard<std::mutex> g(mu_);
            if (!spare_events_.empty()) { hipEvent_t e = spare_events_.back(); spare_events_.pop_back(); return e; }
        }
        hipEvent_t e = nullptr;
        return hipEventCreateWithFlags(&e, hipEventDisableTiming) == hipSuccess ? e : nullptr;
    }
    void give_event(hipEvent_t e) { std::lock_guard<std::mutex> g(mu_); spare_events_.push_back(e); }

    RawAlloc alloc_;
    RawFree free_;
    size_t cap_;
    std::mutex mu_;
    std::map<int, std::multimap<size_t, Block>> free_list_;
    std::unordered_map<void*, Live> live_;
    std::vector<hipEvent_t> spare_events_;
    CacheStats st_;
};

inline size_t env_mb(const char* name, size_t dflt_mb) {
    const char* e = getenv(name);
    if (!e || !e[0]) return dflt_mb << 20;
    const size_t mb = (size_t)strtoull(e, nullptr, 10);
    return mb < 256 ? (size_t)256 << 20 : mb > SIZE_MAX >> 20 ? SIZE_MAX : mb << 20;
}
inline hipError_t raw_dev_alloc(void** p, size_t n) { return hipMalloc(p, n); }
inline hipError_t raw_dev_free(void* p) { return hipFree(p); }
inline BlockCache& dev_cache() {      // (never destroyed: the runtime may already be gone when static destructors run)
    static BlockCache* c = new BlockCache(raw_dev_alloc, raw_dev_free, env_mb("NP_DEVCACHE_MB", 16384));
    return *c;
}


inline hipError_t raw_host_alloc(void** p, size_t n) { return hipHostMalloc(p, n, hipHostMallocPortable); }
inline hipError_t raw_host_free(void* p) { return hipHostFree(p); }
inline BlockCache& host_cache() {
    static BlockCache* c = new BlockCache(raw_host_alloc, raw_host_free, env_mb("NP_PINCACHE_MB", 2048));
    return *c;
}
inline hipError_t host_malloc(void** p, size_t bytes, unsigned /*flags: every block is hipHostMallocPortable*/) {
    const hipError_t e = host_cache().get(p, bytes ? bytes : 1);
    if (e == hipSuccess) {
        alloc_log("H+", *p, bytes);
        PinnedRanges& R = pinned_ranges();
        std::lock_guard<std::mutex> g(R.mu);
        R.live[(uintptr_t)*p] = bytes;
    }
    return e;
}
inline hipError_t host_free(void* p) {
    if (!p) return hipSuccess;
    alloc_log("H-", p, 0);
    {
        PinnedRanges& R = pinned_ranges();
        std::lock_guard<std::mutex> g(R.mu);
        R.live.erase((uintptr_t)p);
    }
    return host_cache().put(p);
}
// What a stopped process can say about itself (tests/conftest.py's watchdog calls np1_diag_report / np2_diag_report from a helper thread):
// every stream of the registry with hipStreamQuery's answer, and the cache counters: whether the stopped thread still has work to wait for.
inline void report(int fd, const char* who) {
    StreamRegistry& R = stream_registry();
    const auto line = [fd](hipStream_t q, int dev) {
        const hipError_t e = hipStreamQuery(q);
        dprintf(fd, "[np diag]   stream %p device %d: %s\n", (void*)q, dev, e == hipSuccess ? "ready" : e == hipErrorNotReady ? "NOT READY" : hipGetErrorString(e));
    };
    std::shared_lock<std::shared_timed_mutex> g(R.mu, std::chrono::seconds(2));
    if (g.owns_lock()) {
        dprintf(fd, "[np diag] %s: %zu stream(s) in the registry (+ the null stream)\n", who, R.live.size());
        for (auto& kv : R.live) line(kv.first, kv.second);
        g.unlock();
    } else dprintf(fd, "[np diag] %s: a thread holds the stream registry\n", who);
    line(nullptr, -1);
    (void)hipGetLastError();
    for (int k = 0; k < 2; ++k) {
        BlockCache& c = k ? host_cache() : dev_cache();
        const CacheStats st = c.stats();
        dprintf(fd, "[np diag]   %s cache (bound %zu MiB): %llu hits, %llu misses, %llu runtime frees, %llu blocks fenced at release, %llu skipped not ready, %llu flushes; "
                    "%zu MiB idle now (peak %zu), %zu MiB handed out\n",
                k ? "pinned-host" : "device", c.cap() >> 20, (unsigned long long)st.hits, (unsigned long long)st.misses, (unsigned long long)st.raw_frees,
                (unsigned long long)st.fenced, (unsigned long long)st.not_ready, (unsigned long long)st.flushes, st.cached >> 20, st.peak_cached >> 20, st.live >> 20);
    }
}

inline int poison() {      // -1: off
    static const int v = [] {
        const char* e = getenv("NP_DEVPOISON");
        if (!e || !e[0] || !strcmp(e, "0")) return -1;
        if (!strcmp(e, "1") || !strcmp(e, "2")) return 0xa5;
        return (int)(strtol(e, nullptr, 16) & 0xff);
    }();
    return v;
}

inline bool poison_runs() {      // NP_DEVPOISON=2: also the work buffers of a batch before every run (np1_batch::poison_work)
    static const bool on = [] { const char* e = getenv("NP_DEVPOISON"); return poison() >= 0 && e && !strcmp(e, "2"); }();
    return on;
}

inline hipError_t dev_malloc(void** p, size_t bytes) {
    const hipError_t e = dev_cache().get(p, bytes);
    if (e == hipSuccess) alloc_log("D+", *p, bytes);
    if (e == hipSuccess && poison() >= 0 && bytes) {
        (void)hipMemsetAsync(*p, poison(), bytes, nullptr);
        (void)hipStreamSynchronize(nullptr);
    }
    return e;
}

inline hipError_t dev_free(void* p) {
    if (!p) return hipSuccess;
    alloc_log("D-", p, 0);
    return dev_cache().put(p);
}

}  // namespace npalloc
