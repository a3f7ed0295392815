// Compiled and run by test_once_per_device.py: which GPUs are asked, and when.
#include <cstdio>

#include "hip_status.h"

static spmm::engine::OncePerDevice once;

static int asked(int device, hipError_t answer, hipError_t want) {
    int calls = 0;
    const hipError_t got = once.on(device, [&] {
        ++calls;
        return answer;
    });
    return got == want ? calls : -1;
}

int main() {
    const hipError_t ok = hipSuccess, bad = hipErrorInvalidValue;
    const bool right = asked(0, bad, bad) == 1 &&  // a failure is told
                       asked(0, ok, ok) == 1 &&    // and not kept
                       asked(0, bad, ok) == 0 &&   // done there
                       asked(1, ok, ok) == 1 &&    // another GPU is asked for itself
                       asked(1, ok, ok) == 0 && asked(0, ok, ok) == 0 &&
                       asked(1000, ok, ok) == 1 && asked(1000, bad, bad) == 1;
    std::puts(right ? "right" : "wrong");
    return right ? 0 : 1;
}
