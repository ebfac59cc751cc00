// What the translation units behind the C ABI share: the error message of the calling thread, the check of a HIP call,
// and a guard that leaves the caller's current device as it was.
#pragma once
#include <hip/hip_runtime.h>

#include <string>

namespace mppi {
// stores the message mppi_last_error() returns on this thread; gives the code back
__attribute__((visibility("hidden"))) int fail(int code, const std::string& msg);

struct DeviceGuard {
    int before = -1;
    hipError_t enter(int device) {
        const hipError_t e = hipGetDevice(&before);
        if (e != hipSuccess) { before = -1; return e; }
        if (before == device) { before = -1; return hipSuccess; }
        return hipSetDevice(device);
    }
    ~DeviceGuard() { if (before >= 0) (void)hipSetDevice(before); }
};
}  // namespace mppi

#define HIP_OK(expr)                                                                                   \
    do {                                                                                               \
        hipError_t e_ = (expr);                                                                        \
        if (e_ != hipSuccess)                                                                          \
            return mppi::fail(-2, std::string(#expr) + ": " + hipGetErrorString(e_));                  \
    } while (0)
