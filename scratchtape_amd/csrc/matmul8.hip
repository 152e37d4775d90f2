// Products of 8-bit rows and 8-bit weights (quant8.h): out[i, j] = (sum over l of x[i, l] w[j, l]) xs[i] ws[j] + bias[j], then
// ReLU; and the gated form act(gate) up of two such products.  Sums of codes are exact in 32-bit integers (k <= 131072:
// 128 x 128 x 131072 = 2^31 is passed by no sum of codes up to 127, and reached only by -128 throughout); the scales enter once, in f32.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "lanes.h"
#include "quant4.h"

namespace {

typedef int32_t i4 __attribute__((ext_vector_type(4)));
typedef int32_t i16 __attribute__((ext_vector_type(16)));

struct Product {
    const int8_t *x, *w;
    const float *xs, *ws, *bias;
    int64_t m, k, n, x_stride, w_stride, out_stride;  // n: columns of out; a gated product has 2 n rows of w
    void *out;
    int32_t act;  // ST_ACT_NONE, _RELU, or a gated product's _SILU, _GELU
};

// gate act'd: silu is g / (1 + exp(-g)), gelu g Phi(g) = g / 2 erfc(-g / sqrt 2) (which keeps its digits far below zero).
__device__ __forceinline__ float gated(float g, float u, int32_t act) {
    const float a = act == ST_ACT_SILU ? g / (1.f + __expf(-g)) : 0.5f * g * erfcf(-0.70710678f * g);
    return a * u;
}

__device__ __forceinline__ float scaled(int32_t sum, float xs, float ws, float bias) { return __builtin_fmaf((float)sum * xs, ws, bias); }

// 16 codes from p on, of which `left` are inside the row; unaligned rows are read a byte at a time.
__device__ __forceinline__ i4 load16(const int8_t *p, int64_t left, bool vec) {
    uint32_t v[4] = {0, 0, 0, 0};
    if (vec && left >= 16) return *(const i4 *)p;
#pragma unroll
    for (int i = 0; i < 16; i++)
        if (i < left) v[i >> 2] |= (uint32_t)(uint8_t)p[i] << (8 * (i & 3));
    return i4{(int)v[0], (int)v[1], (int)v[2], (int)v[3]};
}

// Any strides and alignment: 64 rows of x by 64 rows of weights a workgroup, 32 x 32 a wave; a gated product's 64 are 32 of the
// gate's and the same 32 of the other half's.
template <class T, bool GATED>
__global__ __launch_bounds__(256) void k_product8_any(Product a, int64_t tiles_n, bool vec) {
    constexpr int BK = 64, PITCH = BK + 16;
    __shared__ __attribute__((aligned(16))) int8_t lx[64 * PITCH], lw[64 * PITCH];
    __shared__ int32_t sums[64][65];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t m0 = blockIdx.x / tiles_n * 64, n0 = blockIdx.x % tiles_n * (GATED ? 32 : 64);
    const int r = tid >> 2, c = (tid & 3) * 16;
    const int64_t xr = m0 + r, wr = GATED ? n0 + (r & 31) : n0 + r;
    const bool x_in = xr < a.m, w_in = wr < a.n;
    const int8_t *const xp = a.x + (x_in ? xr * a.x_stride : 0) + c;
    const int8_t *const wp = a.w + (w_in ? (wr + (GATED && r >= 32 ? a.n : 0)) * a.w_stride : 0) + c;
    i16 acc;
#pragma unroll
    for (int e = 0; e < 16; e++) acc[e] = 0;
    for (int64_t k0 = 0; k0 < a.k; k0 += BK) {
        const int64_t left = a.k - k0 - c;
        const i4 xv = load16(xp + k0, x_in ? left : 0, vec), wv = load16(wp + k0, w_in ? left : 0, vec);
        __syncthreads();
        *(i4 *)(lx + r * PITCH + c) = xv;
        *(i4 *)(lw + r * PITCH + c) = wv;
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const int at = (lane & 31) * PITCH + s * 32 + (lane >> 5) * 16;
            const i4 xf = *(const i4 *)(lx + (wave >> 1) * 32 * PITCH + at), wf = *(const i4 *)(lw + (wave & 1) * 32 * PITCH + at);
            acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(xf, wf, acc, 0, 0, 0);
        }
    }
#pragma unroll
    for (int e = 0; e < 16; e++) sums[(wave >> 1) * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)][(wave & 1) * 32 + (lane & 31)] = acc[e];
    __syncthreads();
    constexpr int COLUMNS = GATED ? 32 : 64;
    for (int i = tid; i < 64 * COLUMNS; i += 256) {
        const int row = i / COLUMNS, col = i % COLUMNS;
        const int64_t mi = m0 + row, ni = n0 + col;
        if (mi >= a.m || ni >= a.n) continue;
        float y = scaled(sums[row][col], a.xs[mi], a.ws[ni], a.bias ? a.bias[ni] : 0.f);
        if constexpr (GATED)
            y = gated(y, scaled(sums[row][col + 32], a.xs[mi], a.ws[a.n + ni], a.bias ? a.bias[a.n + ni] : 0.f), a.act);
        else if (a.act == ST_ACT_RELU && y < 0.f)
            y = 0.f;
        ((T *)a.out)[mi * a.out_stride + ni] = (T)y;
    }
}

st_status product8(const char *name, const Product &a, int32_t dtype, bool is_gated, const void *work, int64_t work_bytes, st_stream stream) {
    if (a.m < 0 || a.k <= 0 || a.n < 0 || a.k > 131072)
        return st::fail(ST_ERR_INVALID, "%s: m %lld, k %lld (1 to 131072), n %lld", name, (long long)a.m, (long long)a.k, (long long)a.n);
    const int64_t columns = is_gated ? 32 : 64;
    if (a.m > (int64_t)1 << 30 || a.n > (int64_t)1 << 30 || (a.m + 63) / 64 * ((a.n + columns - 1) / columns) >= (int64_t)1 << 24)
        return st::fail(ST_ERR_INVALID, "%s: %lld x %lld outputs are too many for one call", name, (long long)a.m, (long long)a.n);
    if (a.x_stride < a.k || a.w_stride < a.k || a.out_stride < a.n)
        return st::fail(ST_ERR_INVALID, "%s: rows of %lld, %lld and %lld elements lie %lld, %lld and %lld apart", name, (long long)a.k, (long long)a.k,
                        (long long)a.n, (long long)a.x_stride, (long long)a.w_stride, (long long)a.out_stride);
    if (dtype < ST_F32 || dtype > ST_BF16) return st::fail(ST_ERR_INVALID, "%s: dtype %d is none of ST_F32, ST_F16, ST_BF16", name, (int)dtype);
    if (is_gated ? a.act != ST_ACT_SILU && a.act != ST_ACT_GELU : a.act != ST_ACT_NONE && a.act != ST_ACT_RELU)
        return st::fail(ST_ERR_INVALID, "%s: activation %d", name, (int)a.act);
    if (a.m == 0 || a.n == 0) return ST_OK;
    if (!a.x || !a.w || !a.xs || !a.ws || !a.out) return st::fail(ST_ERR_INVALID, "%s: NULL buffer", name);
    const int64_t size = st::dtype_size(dtype);
    if (((uintptr_t)a.out & (size - 1)) || (((uintptr_t)a.xs | (uintptr_t)a.ws | (uintptr_t)a.bias) & 3) || ((uintptr_t)work & 15))
        return st::fail(ST_ERR_INVALID, "%s: a buffer is not aligned to its elements (work: 16 bytes)", name);
    if (!st::device_ok()) return ST_ERR_NO_DEVICE;
    const bool vec = (((uintptr_t)a.x | (uintptr_t)a.w) & 15) == 0 && (a.m == 1 || a.x_stride % 16 == 0) && (a.w_stride % 16 == 0 || (a.n == 1 && !is_gated));
    return st::with_dtype(dtype, [&](auto *t) -> st_status {
        using T = std::remove_pointer_t<decltype(t)>;
        const int64_t tiles_n = (a.n + columns - 1) / columns, tiles = (a.m + 63) / 64 * tiles_n;
        if (is_gated)
            k_product8_any<T, true><<<(uint32_t)tiles, 256, 0, st::stream_of(stream)>>>(a, tiles_n, vec);
        else
            k_product8_any<T, false><<<(uint32_t)tiles, 256, 0, st::stream_of(stream)>>>(a, tiles_n, vec);
        ST_LAUNCH_CHECK();
        return ST_OK;
    });
}

}  // namespace

extern "C" int64_t st_matmul_8bit_bytes(int64_t m, int64_t k, int64_t n, int32_t is_gated) { return 0; }

extern "C" st_status st_matmul_8bit(const int8_t *x, const float *x_scales, int64_t m, int64_t k, int64_t x_stride, const int8_t *w,
                                    const float *w_scales, int64_t n, int64_t w_stride, const float *bias, int32_t relu, void *out, int32_t dtype,
                                    int64_t out_stride, void *work, int64_t work_bytes, st_stream stream) {
    st::clear_error();
    const Product a = {x, w, x_scales, w_scales, bias, m, k, n, x_stride, w_stride, out_stride, out, relu ? ST_ACT_RELU : ST_ACT_NONE};
    return product8("matmul_8bit", a, dtype, false, work, work_bytes, stream);
}

extern "C" st_status st_gated_8bit(const int8_t *x, const float *x_scales, int64_t m, int64_t k, int64_t x_stride, const int8_t *w,
                                   const float *w_scales, int64_t n, int64_t w_stride, const float *bias, int32_t activation, void *out, int32_t dtype,
                                   int64_t out_stride, void *work, int64_t work_bytes, st_stream stream) {
    st::clear_error();
    const Product a = {x, w, x_scales, w_scales, bias, m, k, n, x_stride, w_stride, out_stride, out, activation};
    return product8("gated_8bit", a, dtype, true, work, work_bytes, stream);
}
