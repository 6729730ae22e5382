// lrn_common.h — what the translation units of include/learner_ops.h share: errors, the device guard, element types.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/learner_ops.h"

namespace lrn {

char* error_text();                       // thread-local, 512 bytes (learner_rows.hip)

inline int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(error_text(), 512, fmt, ap);
    va_end(ap);
    return code;
}

// The calling thread's device for the length of a call: a launch goes to the current device, and the stream is `device`'s.
struct DeviceGuard {
    int previous = -1;
    hipError_t err;
    explicit DeviceGuard(int device) {
        err = hipGetDevice(&previous);
        if (err == hipSuccess && previous != device) err = hipSetDevice(device);
        else previous = -1;
    }
    ~DeviceGuard() { if (previous >= 0) (void)hipSetDevice(previous); }
};

#define LRN_ON_DEVICE(device)                                                                                     \
    lrn::DeviceGuard guard_(device);                                                                              \
    if (guard_.err != hipSuccess) return lrn::fail(-2, "device %d: %s", (int)(device), hipGetErrorString(guard_.err))

// A launch that was refused says so through the error of its own call, not of a later one.
#define LRN_LAUNCHED(what)                                                                                        \
    do {                                                                                                          \
        hipError_t err_ = hipGetLastError();                                                                      \
        if (err_ != hipSuccess) return lrn::fail(-4, "%s: %s", what, hipGetErrorString(err_));                    \
    } while (0)

typedef __bf16 bf16;
typedef _Float16 f16;

template <class T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }

constexpr float kNegInf = -__builtin_inff();
constexpr double kLog2e = 1.4426950408889634;

// exp(x) = 2^(x log2 e) on the exponential unit.  log2 e in two parts, so that only the product's rounding counts (relative error of
// the result at most |x| 2^-24 + 1 unit; with the rounded constant alone 1.23 |x| 2^-24): the weights below are exp(z - max), where
// a large |x| is a small weight.  (The low part is positive: -inf stays -inf.)
constexpr float kLog2eHigh = (float)kLog2e, kLog2eLow = (float)(kLog2e - (double)kLog2eHigh);
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(__builtin_fmaf(x, kLog2eHigh, x * kLog2eLow)); }

// log(s) of a sum of weights (1 <= s, or 0: -inf) on the logarithm unit, 1 unit and one rounding off; 1 / s likewise.
__device__ __forceinline__ float fast_log(float s) { return __builtin_amdgcn_logf(s) * 0.6931471805599453f; }
__device__ __forceinline__ float fast_inverse(float s) { return __builtin_amdgcn_rcpf(s); }

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace lrn
