// The 8-bit format of rows of weights and of activations (rms.hip makes it, matmul8.hip multiplies it), and loads and
// stores of eight neighbouring elements.
//
// A row x has a = max |x| and scale = f32(a / 127); value i is held as code = round_half_even(127 x / a), 0 where a = 0,
// and stands for scale * code.  The quotient is decided in 64 bits, so that a value next to the border of two codes has one
// answer whatever computes it.  A row that holds a NaN or an infinity has scale NaN and codes 0.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "common.h"
#include "lanes.h"
#include "quant4.h"

namespace st {

// Eight elements that need the alignment of one: a 16-byte load may begin at any element.
template <class T>
struct Eight {
    typedef T type __attribute__((ext_vector_type(8), aligned(alignof(T))));
};
template <class T>
using Eight_t = typename Eight<T>::type;

template <class T>
struct Parts {
    typedef T two __attribute__((ext_vector_type(2), aligned(alignof(T))));
    typedef T four __attribute__((ext_vector_type(4), aligned(alignof(T))));
};

// Elements at .. at + 7 of a row of `width`, 0 past its end: the row's last ones in a four, a two and a one, whose loads do not wait
// for one another (the norm of 30000 x 1111 f16 into 8 bits 127 us, 161 one by one; of 1112, which has no such end, 103 and 97).
template <class T>
__device__ __forceinline__ Eight_t<T> load_eight(const T *row, int64_t at, int64_t width) {
    typedef typename Parts<T>::two Two;
    typedef typename Parts<T>::four Four;
    if (at + 8 <= width) return *(const Eight_t<T> *)(row + at);
    Eight_t<T> v = {};
    if (at >= width) return v;
    const int left = (int)(width - at);
    const bool has4 = left & 4, has2 = left & 2;
    Four four = {};
    Two two = {}, one = {};
    if (has4) four = *(const Four *)(row + at);
    if (has2) two = *(const Two *)(row + at + (left & 4));
    if (left & 1) one[0] = row[at + (left & 6)];
    const Two behind = has2 ? two : one, last = has2 ? one : Two{};
#pragma unroll
    for (int i = 0; i < 2; i++) {
        v[i] = has4 ? four[i] : behind[i], v[2 + i] = has4 ? four[2 + i] : last[i];
        v[4 + i] = has4 ? behind[i] : T(0), v[6 + i] = has4 ? last[i] : T(0);
    }
    return v;
}

// The same of 16-bit elements in two steps, so that a row's end waits for no load: the load, of the row's last eight where fewer are
// left, and (settle) their move to where they belong, zeros behind them.
template <class T>
__device__ __forceinline__ Eight_t<T> load_raw(const T *row, int64_t at, int64_t width) {
    if (width < 8) return load_eight(row, at, width);
    Eight_t<T> v = {};
    if (at < width) v = *(const Eight_t<T> *)(row + min(at, width - 8));
    return v;
}

template <class T>
__device__ __forceinline__ void settle(Eight_t<T> &v, int64_t at, int64_t width) {
    static_assert(sizeof(T) == 2, "two elements a word");
    typedef uint32_t U4 __attribute__((ext_vector_type(4)));
    const int64_t by = at + 8 - width;  // places to move down
    if (width < 8 || by <= 0 || by >= 8) return;
    U4 u = __builtin_bit_cast(U4, v);
    if (by & 4) u = U4{u[2], u[3], 0, 0};
    if (by & 2) u = U4{u[1], u[2], u[3], 0};
    if (by & 1)
        u = U4{__builtin_amdgcn_alignbit(u[1], u[0], 16), __builtin_amdgcn_alignbit(u[2], u[1], 16), __builtin_amdgcn_alignbit(u[3], u[2], 16), u[3] >> 16};
    v = __builtin_bit_cast(Eight_t<T>, u);
}

template <class T>
__device__ __forceinline__ void store_eight(T *row, int64_t at, int64_t width, Eight_t<T> v) {
    typedef typename Parts<T>::two Two;
    typedef typename Parts<T>::four Four;
    if (at + 8 <= width) {
        *(Eight_t<T> *)(row + at) = v;
        return;
    }
    if (at >= width) return;
    const int left = (int)(width - at);
    const bool has4 = left & 4, has2 = left & 2;
    if (has4) *(Four *)(row + at) = Four{v[0], v[1], v[2], v[3]};
    const Two behind = has4 ? Two{v[4], v[5]} : Two{v[0], v[1]}, last = has4 ? Two{v[6], v[7]} : Two{v[2], v[3]};
    if (has2) *(Two *)(row + at + (left & 4)) = behind;
    if (left & 1) row[at + (left & 6)] = has2 ? last[0] : behind[0];
}

// Codes of eight values t of a row with a = max |t| (finite), in 64 bits.
//
// f32 does as long as it leaves no doubt: t (127 / a) in f32 is off by no more than four roundings (t, a, 127 / a, the product)
// of a number up to 127, 4 x 127 x 2^-24 = 3.03e-5, so a quotient more than 3.2e-5 from the middle of two codes has the code
// that 64 bits give it.  A wave that has one nearer, or an `a` whose quotients could leave f32's normal numbers, divides in 64.
struct RowCodes {
    double a;
    float f;
    bool plain;
    __device__ __forceinline__ explicit RowCodes(double a_) : a(a_), f(127.f / (float)a_), plain(a_ > 0x1p-100 && a_ < 0x1p100) {}

    __device__ __forceinline__ uint2 operator()(const double (&t)[8]) const {
        int c[8];
        float off[8], nearest = 0.5f;  // the distances from the middle of two codes, the least of them
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float r = (float)t[i] * f, n = __builtin_rintf(r);
            off[i] = 0.5f - __builtin_fabsf(r - n);
            nearest = fminf(nearest, off[i]);
            c[i] = (int)n;
        }
        if (!plain || !(nearest > 3.2e-5f)) {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (!plain || !(off[i] > 3.2e-5f)) c[i] = a > 0.0 ? (int)__builtin_rint(t[i] * 127.0 / a) : 0;
        }
        uint2 out = make_uint2(0, 0);
#pragma unroll
        for (int i = 0; i < 4; i++) out.x |= (uint32_t)(c[i] & 255) << (8 * i), out.y |= (uint32_t)(c[4 + i] & 255) << (8 * i);
        return out;
    }
};

// The largest finite number of a type.
template <class T>
__device__ constexpr float largest() { return sizeof(T) == 4 ? 0x1.fffffep127f : std::is_same_v<T, _Float16> ? 65504.f : 0x1.fep127f; }

// What code i (0 .. 7) of eight stands for, no larger than T holds: 127 f32(a / 127) can pass an `a` at the end of the range.
template <class T>
__device__ __forceinline__ T code_value(uint2 codes, int i, float scale) {
    const float v = (float)(int8_t)((i < 4 ? codes.x : codes.y) >> (8 * (i & 3))) * scale;
    return (T)(__builtin_fabsf(v) > largest<T>() ? __builtin_copysignf(largest<T>(), v) : v);
}

}  // namespace st
