// A hipMalloc that fails from a size on, for a process that loads it (globally) before the library under test:
// malloc_fails_from(real, bytes) sets the function behind it and the size (0: none fails), malloc_failures() counts.
#include <cstddef>

extern "C" {
static int (*g_real)(void **, size_t) = nullptr;
static size_t g_from = 0;
static long g_failures = 0;

void malloc_fails_from(int (*real)(void **, size_t), size_t bytes) {
    g_real = real;
    g_from = bytes;
}
long malloc_failures() { return g_failures; }

int hipMalloc(void **p, size_t n) {
    if (g_from && n >= g_from) {
        g_failures++;
        return 2;  // hipErrorOutOfMemory
    }
    return g_real(p, n);
}
}
