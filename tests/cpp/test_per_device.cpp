// OncePerDevice (csrc/per_device.h) on a stand-in for the runtime's current device: once on every device,
// again after a failure, and never on the word of another device.
#include <cstdio>

#include "per_device.h"

static int current = 0;
static cudaError_t answer = cudaSuccess;
extern "C" cudaError_t cudaGetDevice(int* dev) {
    *dev = current;
    return answer;
}

static int failures = 0;
#define CHECK(c)                                                 \
    do {                                                         \
        if (!(c)) {                                              \
            std::printf("line %d: %s\n", __LINE__, #c);          \
            ++failures;                                          \
        }                                                        \
    } while (0)

int main() {
    g4b::OncePerDevice once;
    int runs = 0;
    const auto good = [&] { return ++runs, cudaSuccess; };
    const auto bad = [&] { return ++runs, cudaErrorInvalidValue; };
    CHECK(once(good) == cudaSuccess && once(good) == cudaSuccess && runs == 1);
    current = 7;
    CHECK(once(bad) == cudaErrorInvalidValue && once(good) == cudaSuccess && once(good) == cudaSuccess && runs == 3);
    current = 63;
    CHECK(once(good) == cudaSuccess && runs == 4);
    current = 0;
    CHECK(once(good) == cudaSuccess && runs == 4);
    current = 64;
    CHECK(once(good) == cudaSuccess && once(good) == cudaSuccess && runs == 6);
    answer = cudaErrorNoDevice;
    CHECK(once(good) == cudaErrorNoDevice && runs == 6);
    return failures;
}
