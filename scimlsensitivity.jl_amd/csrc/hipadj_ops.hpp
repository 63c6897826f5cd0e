// hipadj_ops.hpp — host side shared by the operators without a handle (recurrence, orthogonalised update): the message of a failure, the device of a call.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdio>
#include <tuple>
#include "../../include/hipadj.h"

void ops_set_error(const char* text);          // hipadj_api.hip: the text of hipadj_last_error(NULL), per thread

template <class... A> static int ops_fail(int code, const char* format, A... args) {
    char b[512];
    std::snprintf(b, sizeof(b), format, args...);
    ops_set_error(b);
    return code;
}
static inline int ops_fail(int code, const char* text) { ops_set_error(text); return code; }

// A launch whose status is the launch's own: what hipGetLastError holds may be an earlier error of the host program, which stays there for the program to see.
inline thread_local hipError_t ops_status = hipSuccess;                 // first failure of the current call's launches
template <class... P, class... A> static void ops_launch(void (*kernel)(P...), dim3 grid, dim3 block, hipStream_t stream, const A&... a) {
    std::tuple<P...> p(a...);
    std::apply([&](P&... q) {
        void* args[] = {(void*)&q...};
        const hipError_t e = hipLaunchKernel((const void*)kernel, grid, block, args, 0, stream);
        if (ops_status == hipSuccess) ops_status = e;
    }, p);
}

// makes `device` current for the duration of a call and the caller's device current again afterwards
struct OpsDevice {
    int rc = HIPADJ_OK, old = -1;
    explicit OpsDevice(int device) {
        ops_status = hipSuccess;
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
    if (ops_status == hipSuccess) return HIPADJ_OK;
    (void)hipGetLastError();                        // this call reports it
    return ops_fail(HIPADJ_ERR_HIP, "%s: %s", what, hipGetErrorString(ops_status));
}
