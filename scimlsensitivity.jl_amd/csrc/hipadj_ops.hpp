// hipadj_ops.hpp — host side shared by the operators without a handle (recurrence, orthogonalised update): the message of a failure, the device of a call.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdio>
#include "../../include/hipadj.h"

void ops_set_error(const char* text);          // hipadj_api.hip: the text of hipadj_last_error(NULL), per thread

template <class... A> static int ops_fail(int code, const char* format, A... args) {
    char b[512];
    std::snprintf(b, sizeof(b), format, args...);
    ops_set_error(b);
    return code;
}
static inline int ops_fail(int code, const char* text) { ops_set_error(text); return code; }

// makes `device` current for the duration of a call and the caller's device current again afterwards
struct OpsDevice {
    int rc = HIPADJ_OK, old = -1;
    explicit OpsDevice(int device) {
        (void)hipGetLastError();                    // of an earlier call of the host program: ops_launched reports this call's launches
        int n = 0;
        if (hipGetDeviceCount(&n) != hipSuccess || n <= 0) { (void)hipGetLastError(); rc = ops_fail(HIPADJ_ERR_NO_DEVICE, "no usable HIP device (gfx950 required; there is no CPU fallback)"); return; }
        if (device < 0 || device >= n) { rc = ops_fail(HIPADJ_ERR_INVALID_ARG, "device %d out of range (%d visible)", device, n); return; }
        int cur = 0;
        if (hipGetDevice(&cur) != hipSuccess) { rc = ops_fail(HIPADJ_ERR_HIP, "hipGetDevice failed"); return; }
        if (cur != device) {
            if (hipSetDevice(device) != hipSuccess) { rc = ops_fail(HIPADJ_ERR_HIP, "hipSetDevice(%d) failed", device); return; }
            old = cur;
        }
    }
    ~OpsDevice() { if (old >= 0) (void)hipSetDevice(old); }
};

// a refused launch (bad grid, no code object for the device) is a status of the call that made it
static inline int ops_launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? HIPADJ_OK : ops_fail(HIPADJ_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}
