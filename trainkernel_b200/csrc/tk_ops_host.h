// Host-side helpers shared by the translation units of libtrainkernel_ops.so: error text, device scope, launch count.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "trainkernel_ops.h"

namespace tk_ops {

int fail(int code, const char* format, ...);
int check(cudaError_t status, const char* what);
void count_launch();
int sm_count(int device);            // multiprocessors, remembered per device; 0 when the device cannot be asked

// Makes `device` current for the calls in its scope and puts the previous one back.  The previous device is
// only ever re-selected, never a device this process has not used.
struct DeviceScope {
    int previous = -1;
    bool switched = false;
    int status = 0;
    explicit DeviceScope(int device) {
        cudaError_t result = cudaGetDevice(&previous);
        if (result == cudaSuccess && previous != device) {
            result = cudaSetDevice(device);
            switched = result == cudaSuccess;
        }
        status = check(result, "selecting the device");
    }
    ~DeviceScope() {
        if (switched) cudaSetDevice(previous);
    }
};

}  // namespace tk_ops
