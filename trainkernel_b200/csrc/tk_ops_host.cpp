// Error text, launch count and device facts of libtrainkernel_ops.so (see include/trainkernel_ops.h).
#include "tk_ops_host.h"

#include <cstdarg>
#include <cstdio>

namespace {
thread_local char g_error[512] = "";
std::atomic<uint64_t> g_launches{0};
constexpr int kMaxDevices = 64;
std::atomic<int> g_sm_count[kMaxDevices];
}  // namespace

namespace tk_ops {

int fail(int code, const char* format, ...) {
    va_list args;
    va_start(args, format);
    vsnprintf(g_error, sizeof(g_error), format, args);
    va_end(args);
    return code;
}

int check(cudaError_t status, const char* what) {
    if (status == cudaSuccess) return 0;
    cudaGetLastError();                            // reported here and now: it must not be taken for a later call's
    return fail(static_cast<int>(status), "trainkernel: %s failed: %s", what, cudaGetErrorString(status));
}

void count_launch() { g_launches.fetch_add(1, std::memory_order_relaxed); }

int sm_count(int device) {
    if (device < 0 || device >= kMaxDevices) return 0;
    int known = g_sm_count[device].load(std::memory_order_relaxed);
    if (!known) {
        if (cudaDeviceGetAttribute(&known, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return 0;
        g_sm_count[device].store(known, std::memory_order_relaxed);
    }
    return known;
}

}  // namespace tk_ops

extern "C" const char* tk_ops_last_error(void) { return g_error; }
extern "C" uint64_t tk_ops_launch_count(void) { return g_launches.load(std::memory_order_relaxed); }
