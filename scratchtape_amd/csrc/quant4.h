// The 4-bit format of the quantised weights (quant4.hip) and of the paged cache (kv4.hip), and the loads and
// stores of the three element types that both take.
//
// A group of values x has lo = min x, hi = max x (f32) and scale = f32((hi - lo) / 15); value i is held as
// code = round_half_even((x - lo) * 15 / (hi - lo)), 0 where hi = lo, and stands for scale * code + lo.  The
// difference, the product and the quotient are taken in 64 bits, so that a value next to the border of two codes has
// one answer whatever computes it.  A group that holds a NaN or an infinity has scale = lo = NaN and codes 0: every
// value of it is NaN.  Code i is at byte i / 2, bits 4 (i % 2); a group's scale and lo are side by side (float2).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.h"
#include "lanes.h"

namespace st {

// Eight consecutive elements as f32.  vec: p is 16-byte aligned (8-byte pairs suffice for no type, so this is asked for
// as a whole); otherwise element by element.
__device__ __forceinline__ void load8(const float *p, bool vec, float (&x)[8]) {
    if (vec) {
        const float4 a = ((const float4 *)p)[0], b = ((const float4 *)p)[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = p[i];
    }
}

template <class T>  // _Float16, __bf16
__device__ __forceinline__ void load8(const T *p, bool vec, float (&x)[8]) {
    typedef T T8 __attribute__((ext_vector_type(8)));
    if (vec) {
        const T8 a = *(const T8 *)p;
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (float)a[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (float)p[i];
    }
}

__device__ __forceinline__ void store8(float *p, bool vec, const float (&x)[8]) {
    if (vec) {
        ((float4 *)p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        ((float4 *)p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = x[i];
    }
}

template <class T>
__device__ __forceinline__ void store8(T *p, bool vec, const float (&x)[8]) {
    typedef T T8 __attribute__((ext_vector_type(8)));
    if (vec) {
        T8 a;
#pragma unroll
        for (int i = 0; i < 8; i++) a[i] = (T)x[i];  // round to nearest even
        *(T8 *)p = a;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = (T)x[i];
    }
}

// The 4-bit form of a group spread over LANES neighbouring lanes (a power of two up to 64, the group starting at a
// multiple of it), 8 values x a lane; lanes with used = false hold none of it.  Returns the lane's 8 codes, and scale
// and lo, the same in every lane.  All lanes of the wave take part.
template <int LANES>
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], bool used, float &scale, float &lo) {
#pragma clang fp contract(off)
    const int lane = lane_id();
    float mn = INFINITY, mx = -INFINITY;
    bool finite = true;
    if (used) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            mn = fminf(mn, x[i]);
            mx = fmaxf(mx, x[i]);
            finite = finite && __builtin_isfinite(x[i]);
        }
    }
    mn = finite ? mn : -INFINITY;  // a value that is not finite shows in the group's minimum
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) {
        mn = fminf(mn, xor_lane(mn, o, lane));
        mx = fmaxf(mx, xor_lane(mx, o, lane));
    }
    const double d = (double)mx - (double)mn;
    if (mn == -INFINITY) {
        scale = lo = NAN;
        return 0;
    }
    scale = (float)(d / 15.0);
    lo = mn;
    if (!(d > 0.0)) return 0;
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) codes |= (uint32_t)(int)rint((((double)x[i] - (double)mn) * 15.0) / d) << (4 * i);
    return codes;
}

// What 8 codes of a group stand for.
__device__ __forceinline__ void values8(uint32_t codes, float scale, float lo, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = __builtin_fmaf(scale, (float)((codes >> (4 * i)) & 15), lo);
}

// Calls f with a null pointer of the element type (ST_F32, ST_F16, ST_BF16) and returns what it returns.
template <class F>
inline st_status with_dtype(int32_t dtype, F &&f) {
    switch (dtype) {
        case ST_F32:
            return f((float *)nullptr);
        case ST_F16:
            return f((_Float16 *)nullptr);
        case ST_BF16:
            return f((__bf16 *)nullptr);
        default:
            return fail(ST_ERR_INVALID, "dtype %d is none of ST_F32, ST_F16, ST_BF16", (int)dtype);
    }
}

inline int64_t dtype_size(int32_t dtype) { return dtype == ST_F32 ? 4 : 2; }

// Whether rows of `stride` elements of `size` bytes from p on are each 16-byte aligned.
inline bool rows_aligned(const void *p, int64_t stride, int64_t size) {
    return ((uintptr_t)p & 15) == 0 && ((stride * size) & 15) == 0;
}

}  // namespace st
