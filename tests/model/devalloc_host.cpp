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

int main(int argc, char** argv) {
    const char* what = argc > 1 ? argv[1] : "";
    if (!strcmp(what, "reuse")) return reuse();
    fprintf(stderr, "devalloc_host reuse\n");
    return 2;
}
