// recurrent.h — what the kernels of a recurrent policy share (conv.hip,
// scan.hip, draw.hip, clip.hip): element types, the error text, small
// numerics. Included by those files only.
#ifndef SDFR_RECURRENT_H
#define SDFR_RECURRENT_H

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <type_traits>

#include "../../include/sdfr.h"

inline thread_local char g_rec_err[256];

__attribute__((format(printf, 2, 3))) inline int32_t rec_fail(int32_t code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_rec_err, sizeof g_rec_err, fmt, ap);
    va_end(ap);
    return code;
}

inline int32_t rec_launched(const char* fn) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return rec_fail(-4, "%s: launch failed: %s", fn, hipGetErrorString(e));
    return 0;
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLog2eLow = 1.9259629911266175e-8f;   // log2(e) - (float)log2(e)
constexpr float kLn2 = 0.6931471805599453f;

inline int rec_size(int32_t dtype) { return dtype == SDFR_F32 ? 4 : 2; }
inline bool rec_float(int32_t dtype) { return dtype == SDFR_F32 || dtype == SDFR_F16 || dtype == SDFR_BF16; }

// Calls F with a value of the element type.
template <class F>
inline int32_t rec_typed(int32_t dtype, F f) {
    if (dtype == SDFR_F32) return f((float)0);
    if (dtype == SDFR_F16) return f((_Float16)0);
    return f((__bf16)0);
}

namespace rec {

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }   // one v_exp_f32

// e^x in one v_exp_f32: the product's rounding error and log2(e)'s own go
// into a first-order factor, so the error stays at the instruction's 1 ulp
// for any x (without them it grows with |x|: 3e-7 at x = -7).
__device__ inline float exp_near(float x) {
    const float hi = x * kLog2e;
    const float lo = __builtin_fmaf(x, kLog2eLow, __builtin_fmaf(x, kLog2e, -hi));
    const float e = exp2_fast(hi);
    // beyond v_exp_f32's range hi says it all (and lo may be inf - inf)
    return fabsf(hi) < 150.0f ? __builtin_fmaf(e, lo * kLn2, e) : e;
}

__device__ inline float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + exp2_fast(-x * kLog2e)); }

}  // namespace rec

#endif
