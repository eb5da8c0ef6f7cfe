// np_devalloc.h over the host stand-in of the runtime (hip_host/): devalloc_host <check>; prints one line of counts, the tests read them.
#include <cstdio>
#include <cstring>
#include "np_devalloc.h"

// the same 40 buffers taken and given back 25 times
static int reuse() {
    void* p[40];
    for (int pass = 0; pass < 25; ++pass) {
        for (int i = 0; i < 40; ++i) if (npalloc::dev_malloc(&p[i], 1000 + 70000 * (size_t)i) != hipSuccess) return 1;
        for (int i = 0; i < 40; ++i) (void)npalloc::dev_free(p[i]);
        for (int i = 0; i < 40; ++i) if (npalloc::host_malloc(&p[i], 1000 + 7000 * (size_t)i, 0) != hipSuccess) return 1;
        for (int i = 0; i < 40; ++i) (void)npalloc::host_free(p[i]);
    }
    printf("mallocs %d frees %d host_mallocs %d host_frees %d\n", fake().mallocs.load(), fake().frees.load(), fake().host_mallocs.load(), fake().host_frees.load());
    return 0;
}

// A thread gives memory back (to the cache, or the cache's blocks to the runtime) while another destroys a stream.  Every runtime call takes
// 40 ms, so the releasing thread is still at the first of five streams when the last of them is destroyed.
static int beside_destroy(bool flush) {
    hipStream_t q[5];
    for (auto& s : q) if (npalloc::stream_create(&s) != hipSuccess) return 1;
    void *kept = nullptr, *held = nullptr;
    if (npalloc::dev_malloc(&kept, 4096) != hipSuccess || npalloc::dev_malloc(&held, 4096) != hipSuccess) return 1;
    (void)npalloc::dev_free(kept);
    hipStream_t last = npalloc::stream_registry().live.rbegin()->first;
    for (auto& s : q) s->busy = true;
    fake().slow_ms = 40;
    std::thread releasing([&] { if (flush) npalloc::dev_cache().flush(-1); else (void)npalloc::dev_free(held); });
    while (fake().in_call == 0) std::this_thread::yield();
    (void)npalloc::stream_destroy(last);
    releasing.join();
    printf("used_destroyed %d left %d gone %d\n", fake().used_destroyed.load(), (int)npalloc::stream_registry().live.size(), last->gone ? 1 : 0);
    return 0;
}

int main(int argc, char** argv) {
    const char* what = argc > 1 ? argv[1] : "";
    if (!strcmp(what, "reuse")) return reuse();
    if (!strcmp(what, "free_beside_destroy")) return beside_destroy(false);
    if (!strcmp(what, "flush_beside_destroy")) return beside_destroy(true);
    fprintf(stderr, "devalloc_host reuse|free_beside_destroy|flush_beside_destroy\n");
    return 2;
}
