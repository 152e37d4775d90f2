// 4-bit weights: the quantiser (the format is in quant4.h) and the products of a few rows with them.
#include <algorithm>

#include "common.h"
#include "lanes.h"
#include "quant4.h"

namespace {

// One thread per 8 values; a group is 4, 8 or 16 neighbouring lanes.
template <class T, int GROUP>
__global__ __launch_bounds__(256) void k_quantise4(const T *__restrict__ x, int64_t n, int64_t k, int64_t stride,
                                                   bool vec, uint32_t *__restrict__ codes, float2 *__restrict__ scales,
                                                   T *__restrict__ values, bool vec_values) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, total = n * (k / 8);
    const bool used = i < total;
    float v[8] = {};
    if (used) {
        const int64_t row = i / (k / 8);
        st::load8(x + row * stride + (i - row * (k / 8)) * 8, vec, v);
    }
    float scale, lo;
    const uint32_t c = st::quantise8<GROUP / 8>(v, used, scale, lo);
    if (!used) return;
    codes[i] = c;
    if (i % (GROUP / 8) == 0) scales[i / (GROUP / 8)] = make_float2(scale, lo);
    if (values) {
        st::values8(c, scale, lo, v);
        st::store8(values + i * 8, vec_values, v);
    }
}

// One wave per output: lane l takes every 64th run of 8 weights.
template <class T>
__global__ __launch_bounds__(256) void k_matvec4(const T *__restrict__ x, int64_t m, int64_t k, int64_t x_stride,
                                                 bool vec, const uint32_t *__restrict__ codes,
                                                 const float2 *__restrict__ scales, int64_t group, int64_t n,
                                                 const float *__restrict__ bias, bool relu, T *__restrict__ out,
                                                 int64_t out_stride) {
    const int64_t col = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (col >= n) return;
    for (int64_t row = blockIdx.y; row < m; row += gridDim.y) {
        float acc = 0.f;
        for (int64_t i = lane; i < k / 8; i += 64) {
            float v[8];
            st::load8(x + row * x_stride + i * 8, vec, v);
            const uint32_t c = codes[col * (k / 8) + i];
            const float2 s = scales[col * (k / group) + i * 8 / group];
            float dot = 0.f, sum = 0.f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                dot += v[j] * (float)((c >> (4 * j)) & 15);
                sum += v[j];
            }
            acc += s.x * dot + s.y * sum;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) acc += st::xor_lane(acc, o, lane);
        if (bias) acc += bias[col];
        if (relu && acc < 0.f) acc = 0.f;
        if (lane == 0) out[row * out_stride + col] = (T)acc;
    }
}

}  // namespace

extern "C" st_status st_quantize_4bit(const void *x, int32_t dtype, int64_t n, int64_t k, int64_t x_stride,
                                      int64_t group, uint8_t *codes, float *scales, void *values, st_stream stream) {
    st::clear_error();
    if (n < 0 || k <= 0) return st::fail(ST_ERR_INVALID, "quantize_4bit: n %lld, k %lld", (long long)n, (long long)k);
    if (group != 32 && group != 64 && group != 128)
        return st::fail(ST_ERR_INVALID, "quantize_4bit: group %lld is none of 32, 64, 128", (long long)group);
    if (k % group) return st::fail(ST_ERR_INVALID, "quantize_4bit: k %lld is not a multiple of the group %lld", (long long)k, (long long)group);
    if (x_stride < k) return st::fail(ST_ERR_INVALID, "quantize_4bit: rows of %lld elements lie %lld apart", (long long)k, (long long)x_stride);
    if (n > (((int64_t)1 << 31) - 1) * 256 / (k / 8)) return st::fail(ST_ERR_INVALID, "quantize_4bit: %lld x %lld values are too many for one call", (long long)n, (long long)k);
    if (dtype < ST_F32 || dtype > ST_BF16) return st::fail(ST_ERR_INVALID, "quantize_4bit: dtype %d is none of ST_F32, ST_F16, ST_BF16", (int)dtype);
    if (n == 0) return ST_OK;
    if (!x || !codes || !scales) return st::fail(ST_ERR_INVALID, "quantize_4bit: NULL buffer");
    const int64_t size = st::dtype_size(dtype);
    if (((uintptr_t)x | (uintptr_t)values) & (size - 1)) return st::fail(ST_ERR_INVALID, "quantize_4bit: x or values not aligned to its elements");
    if (((uintptr_t)codes & 3) || ((uintptr_t)scales & 7)) return st::fail(ST_ERR_INVALID, "quantize_4bit: codes are 4-byte, scales 8-byte aligned");
    if (!st::device_ok()) return ST_ERR_NO_DEVICE;
    const bool vec = st::rows_aligned(x, x_stride, size), vec_values = ((uintptr_t)values & 15) == 0;
    const int64_t blocks = (n * (k / 8) + 255) / 256;
    return st::with_dtype(dtype, [&](auto *t) -> st_status {
        using T = std::remove_pointer_t<decltype(t)>;
        auto go = [&](auto kernel) {
            kernel<<<(uint32_t)blocks, 256, 0, st::stream_of(stream)>>>((const T *)x, n, k, x_stride, vec, (uint32_t *)codes,
                                                                        (float2 *)scales, (T *)values, vec_values);
        };
        if (group == 32)
            go(k_quantise4<T, 32>);
        else if (group == 64)
            go(k_quantise4<T, 64>);
        else
            go(k_quantise4<T, 128>);
        ST_LAUNCH_CHECK();
        return ST_OK;
    });
}

extern "C" st_status st_matvec_4bit(const void *x, int32_t dtype, int64_t m, int64_t k, int64_t x_stride,
                                    const uint8_t *codes, const float *scales, int64_t group, int64_t n,
                                    const float *bias, int32_t relu, void *out, int64_t out_stride, st_stream stream) {
    st::clear_error();
    if (m < 0 || k <= 0 || n < 0) return st::fail(ST_ERR_INVALID, "matvec_4bit: m %lld, k %lld, n %lld", (long long)m, (long long)k, (long long)n);
    if (group != 32 && group != 64 && group != 128)
        return st::fail(ST_ERR_INVALID, "matvec_4bit: group %lld is none of 32, 64, 128", (long long)group);
    if (k % group) return st::fail(ST_ERR_INVALID, "matvec_4bit: k %lld is not a multiple of the group %lld", (long long)k, (long long)group);
    if (k > 1 << 20 || m > 1 << 20 || n > (int64_t)1 << 31)
        return st::fail(ST_ERR_INVALID, "matvec_4bit: m %lld, k %lld (up to 2^20 each), n %lld (up to 2^31)", (long long)m, (long long)k, (long long)n);
    if (x_stride < k || out_stride < n)
        return st::fail(ST_ERR_INVALID, "matvec_4bit: rows of %lld and %lld elements lie %lld and %lld apart", (long long)k, (long long)n, (long long)x_stride, (long long)out_stride);
    if (dtype < ST_F32 || dtype > ST_BF16) return st::fail(ST_ERR_INVALID, "matvec_4bit: dtype %d is none of ST_F32, ST_F16, ST_BF16", (int)dtype);
    if (m == 0 || n == 0) return ST_OK;
    if (!x || !codes || !scales || !out) return st::fail(ST_ERR_INVALID, "matvec_4bit: NULL buffer");
    const int64_t size = st::dtype_size(dtype);
    if (((uintptr_t)x | (uintptr_t)out) & (size - 1)) return st::fail(ST_ERR_INVALID, "matvec_4bit: x or out not aligned to its elements");
    if (((uintptr_t)codes & 15) || ((uintptr_t)scales & 7) || ((uintptr_t)bias & 3))
        return st::fail(ST_ERR_INVALID, "matvec_4bit: codes are 16-byte, scales 8-byte, bias 4-byte aligned");
    if (!st::device_ok()) return ST_ERR_NO_DEVICE;
    const bool vec = st::rows_aligned(x, x_stride, size);
    return st::with_dtype(dtype, [&](auto *t) -> st_status {
        using T = std::remove_pointer_t<decltype(t)>;
        k_matvec4<T><<<dim3((uint32_t)((n + 3) / 4), (uint32_t)std::min<int64_t>(m, 65535)), 256, 0, st::stream_of(stream)>>>(
            (const T *)x, m, k, x_stride, vec, (const uint32_t *)codes, (const float2 *)scales, group, n, bias, relu != 0,
            (T *)out, out_stride);
        ST_LAUNCH_CHECK();
        return ST_OK;
    });
}
