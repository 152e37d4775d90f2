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

// Eight consecutive elements as f32.  vec: p is 16-byte aligned, and they are read 16 bytes at a time; else one by one.
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
//
// Quotients by d = hi - lo are products with its reciprocal in 64 bits and one correction, q + (a - q d) / d, which is
// a / d rounded (the reciprocal is).  For the codes f32 does as long as it leaves no doubt: (x - lo) (15 / d) in f32 is off by
// no more than 4 roundings (d, 15 / d, the difference, the product) of a number up to 15, 4 x 15 x 2^-24 = 3.6e-6, so a
// quotient more than 1e-5 from the middle of two codes has the code that 64 bits give it.  Where a wave has one that is nearer
// (or d is so small or so large that these products would leave f32's normal numbers), it computes its codes again in 64.
template <int LANES>
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], bool used, float &scale, float &lo) {
#pragma clang fp contract(off)
    const int lane = lane_id();
    float mn = INFINITY, mx = -INFINITY;
    if (used) {
        float zero = 0.f;  // NaN once a value is not finite
#pragma unroll
        for (int i = 0; i < 8; i++) {
            mn = fminf(mn, x[i]);
            mx = fmaxf(mx, x[i]);
            zero = __builtin_fmaf(x[i], 0.f, zero);
        }
        if (zero != 0.f) mn = -INFINITY;  // which then shows in the group's minimum
    }
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) {
        mn = fminf(mn, xor_lane(mn, o, lane));
        mx = fmaxf(mx, xor_lane(mx, o, lane));
    }
    const bool finite = mn != -INFINITY && used;
    lo = finite ? mn : NAN;
    const double d = finite ? (double)mx - (double)mn : 0.0;
    const double third = d * (1.0 / 15.0);
    const float fifteenth = (float)__builtin_fma(__builtin_fma(-15.0, third, d), 1.0 / 15.0, third);
    scale = finite ? fifteenth : NAN;
    const float f = 15.f / (float)d;  // (d 0: infinite, and not used)
    const bool plain = d > 0x1p-100 && d < 0x1p100;
    uint32_t codes = 0;
    float nearest = 0.5f;  // the least distance from the middle of two codes
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float r = (x[i] - mn) * f, c = __builtin_rintf(r);
        nearest = fminf(nearest, 0.5f - __builtin_fabsf(r - c));
        codes |= (uint32_t)(int)c << (4 * i);
    }
    if (d == 0.0) codes = 0;
    if (d > 0.0 && (!plain || !(nearest > 1e-5f))) {
        const double reciprocal = 1.0 / d;
        codes = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const double a = ((double)x[i] - (double)mn) * 15.0, q = a * reciprocal;
            codes |= (uint32_t)(int)rint(__builtin_fma(__builtin_fma(-q, d, a), reciprocal, q)) << (4 * i);
        }
    }
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
