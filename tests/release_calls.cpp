// Counts the release calls of ts_tensor_from_device and ts_packed8_from_device
// while each allocation of the call in turn fails: one call, whatever happens.
// (Empty tensors and refused ones: no device is touched.)
#include <cstdio>
#include <cstdlib>
#include <new>

#include "ts_gradtrack.h"

static long fail_at = -1;  // allocations until one fails (once); below zero: none does

void *operator new(std::size_t n) {
    if (fail_at >= 0 && fail_at-- == 0) throw std::bad_alloc();
    if (void *p = std::malloc(n ? n : 1)) return p;
    throw std::bad_alloc();
}
void operator delete(void *p) noexcept { std::free(p); }
void operator delete(void *p, std::size_t) noexcept { std::free(p); }

static int calls = 0;
static void released(void *ctx) { calls += ctx == &calls; }

int main() {
    const size_t empty[2] = {0, 3}, wraps[2] = {size_t(1) << 40, size_t(1) << 40};
    int made = 0, bad = 0;
    for (int kind = 0; kind < 4; ++kind) {
        for (long n = -1; n < 24; ++n) {
            calls = 0;
            fail_at = n;
            if (kind < 2) {
                ts_tensor *t = ts_tensor_from_device(nullptr, kind ? wraps : empty, 2, released, &calls);
                fail_at = -1;
                made += t != nullptr;
                ts_tensor_free(t);
            } else {
                ts_packed8 *p = ts_packed8_from_device(nullptr, nullptr, kind == 3 ? size_t(1) << 60 : 0, 128, released, &calls);
                fail_at = -1;
                made += p != nullptr;
                ts_packed8_free(p);
            }
            if (calls != 1) {
                std::printf("kind %d, allocation %ld fails: %d calls\n", kind, n, calls);
                ++bad;
            }
        }
    }
    std::printf("%d made, %d wrong\n", made, bad);
    return made < 2 || bad;
}
