// zq_entry.hpp -- what the C entry points on device pointers share: alignment
// checks, status codes, and the device that a call works on.
#pragma once
#include "../../include/zq_hip.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace zq {

inline bool a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool a4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

inline int status(hipError_t e) { return e == hipSuccess ? ZQ_OK : e == hipErrorInvalidValue ? ZQ_ERR_ARG : ZQ_ERR_HIP; }

// The device that holds the cache made current for the call's launches, and the
// caller's device again after it.
class OnDeviceOf {
public:
    explicit OnDeviceOf(const void* p) {
        hipPointerAttribute_t a;
        if (hipPointerGetAttributes(&a, p) != hipSuccess) {
            (void)hipGetLastError();
            int n = 0;
            st_ = hipGetDeviceCount(&n) == hipSuccess && n > 0 ? ZQ_ERR_ARG : ZQ_ERR_NO_DEVICE;
            (void)hipGetLastError();
            return;
        }
        if (a.type != hipMemoryTypeDevice && a.type != hipMemoryTypeManaged) {
            st_ = ZQ_ERR_ARG;  // an address of the host: a kernel that used it would fault
            return;
        }
        dev_ = a.device;
        if (hipGetDevice(&was_) != hipSuccess) st_ = ZQ_ERR_HIP;
        else if (a.device != was_) {
            moved_ = hipSetDevice(a.device) == hipSuccess;
            if (!moved_) st_ = ZQ_ERR_HIP;
        }
    }
    ~OnDeviceOf() {
        if (moved_) (void)hipSetDevice(was_);
    }
    int status() const { return st_; }
    // p is memory of that device, too
    bool holds(const void* p) const {
        hipPointerAttribute_t a;
        if (hipPointerGetAttributes(&a, p) != hipSuccess) {
            (void)hipGetLastError();
            return false;
        }
        return (a.type == hipMemoryTypeDevice || a.type == hipMemoryTypeManaged) && a.device == dev_;
    }

private:
    int was_ = 0, dev_ = 0, st_ = ZQ_OK;
    bool moved_ = false;
};

}  // namespace zq
