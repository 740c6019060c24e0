// Host threads that raise one kernel's shared-memory limit to different sizes at the
// same time (linked with fake_runtime.cc). The call for the larger size, once it has set
// the limit, is held back in the runtime until the other one is through, or for
// half a second if it does not come. Prints the number of checks that failed.
#include <stdio.h>

#include <atomic>
#include <chrono>
#include <thread>

#include "common.cuh"

static std::atomic<int> limit{48 * 1024}, lowered{0}, calls{0};
static std::atomic<bool> large_is_in{false}, small_is_through{false};
constexpr int LARGE = 200 * 1024, MIDDLE = 150 * 1024, SMALL = 100 * 1024;

extern "C" cudaError_t cudaFuncSetAttribute(const void *, cudaFuncAttribute, int bytes) {
    calls++;
    if (bytes < limit) lowered++;
    limit = bytes;
    if (bytes == LARGE) {
        large_is_in = true;
        for (int i = 0; i < 500 && !small_is_through; i++) std::this_thread::sleep_for(std::chrono::milliseconds(1));
    }
    return cudaSuccess;
}

static void kernel(int) {}

int main() {
    static size_t attr[64];
    std::atomic<int> bad{0};
    std::thread large([&] { bad += ofb::ensure_dyn_smem(kernel, LARGE, attr) != cudaSuccess; });
    while (!large_is_in) std::this_thread::yield();
    std::thread small([&] {
        bad += ofb::ensure_dyn_smem(kernel, SMALL, attr) != cudaSuccess;
        small_is_through = true;
    });
    large.join();
    small.join();
    bad += ofb::ensure_dyn_smem(kernel, MIDDLE, attr) != cudaSuccess;
    bad += limit < MIDDLE;  // what was asked for last must have room
    bad += lowered != 0;
    const int before = calls;
    ofb::ensure_dyn_smem(kernel, LARGE, attr);
    bad += calls != before;  // (the largest is remembered)
    printf("%d\n", bad.load());
    return 0;
}
