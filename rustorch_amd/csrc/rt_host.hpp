// What the files that hold C entries share on the host: error details, the macros around HIP calls and entries, the device.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include <exception>

#include "../../include/rt_attn.h"

#define RT_API extern "C" __attribute__((visibility("default")))

namespace rt {

inline void clear_err(rt_err_detail* e) {
    if (e) {
        e->which = -1;
        e->expected = e->got = e->got2 = 0;
        e->hip_error = 0;
        e->message[0] = 0;
    }
}

inline int fail(rt_err_detail* e, int status, int which, uint64_t expected, uint64_t got, const char* msg, uint64_t got2 = 0) {
    if (e) {
        e->which = which;
        e->expected = expected;
        e->got = got;
        e->got2 = got2;
        e->hip_error = 0;
        snprintf(e->message, sizeof(e->message), "%s", msg ? msg : "");
    }
    return status;
}

inline int fail_hip(rt_err_detail* e, hipError_t code, const char* where) {
    if (e) {
        e->which = -1;
        e->expected = e->got = e->got2 = 0;
        e->hip_error = (int32_t)code;
        snprintf(e->message, sizeof(e->message), "%s: %s", where, hipGetErrorString(code));
    }
    return RT_ERR_HIP;
}

// Finds the gfx950 device on the first call (api.hip); every compute entry calls it behind its own checks.
int ensure_device(rt_err_detail* err);
uint64_t next_launch_id();  // a number no other launch of the process has, its low 8 bits zero

// Does [a, a + n) share a byte with [b, b + m)?
inline bool overlap(const void* a, size_t n, const void* b, size_t m) {
    return n && m && (uintptr_t)a < (uintptr_t)b + m && (uintptr_t)b < (uintptr_t)a + n;
}

}  // namespace rt

#define HIP_TRY(expr, where)                                       \
    do {                                                           \
        hipError_t _e = (expr);                                    \
        if (_e != hipSuccess) return rt::fail_hip(err, _e, where); \
    } while (0)

// Behind the body of an entry that may allocate on the host: no exception passes a C entry.
#define RT_NO_THROW                                               \
    catch (const std::exception& e) {                             \
        return rt::fail_hip(err, hipErrorOutOfMemory, e.what());  \
    }
