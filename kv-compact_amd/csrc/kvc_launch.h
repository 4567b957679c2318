// What the entry points of the paged cache and of its attention share: the
// device of a stream, and launches that report their own error.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/kvc-cache.h"

namespace kvc {

// Makes the stream's device the current one for the length of a call (a
// launch goes to the current device). ok is false when there is no GPU.
struct StreamDevice {
    int was = -1;
    bool moved = false, ok = false;
    explicit StreamDevice(hipStream_t st) {
        if (hipGetDevice(&was) != hipSuccess) {
            (void)hipGetLastError();
            return;
        }
        hipDevice_t dev = was;
        if (st && hipStreamGetDevice(st, &dev) != hipSuccess) {
            (void)hipGetLastError();
            return;
        }
        if (dev != was) {
            if (hipSetDevice(dev) != hipSuccess) {
                (void)hipGetLastError();
                return;
            }
            moved = true;
        }
        ok = true;
    }
    ~StreamDevice() {
        if (moved) (void)hipSetDevice(was);
    }
    StreamDevice(const StreamDevice &) = delete;
    StreamDevice & operator=(const StreamDevice &) = delete;
};

template <class... A>
bool launch(void (*kernel)(A...), dim3 grid, dim3 block, hipStream_t st, A... a) {
    void * args[] = {(void *)&a...};
    if (hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, args, 0, st) == hipSuccess) return true;
    (void)hipGetLastError();
    return false;
}

// 0, or the error of a cache that the calls cannot work on.
int check_cache(const kvc_cache * c);

}  // namespace kvc
