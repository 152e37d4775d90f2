// Appending new tokens to the paged 4-bit cache (kv4.h), with the position rotation of queries and keys.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "kv4.h"
#include "lanes.h"
#include "quant4.h"

namespace {

using st::Cache;
using st::page_of;

struct AppendArgs {
    int64_t n, q_stride, k_stride, v_stride;
    int32_t hq, hd, half, interleaved;
    bool vec_q, vec_k, vec_v, vec_out;
    const int32_t *seq, *pos;
    const float *inv_freq;
    uint8_t *k_codes, *v_codes;
    float2 *k_scales, *v_scales;
    Cache cache;
};

// 8 components from e of a vector, the first 2 half of them rotated by the position's angles in 64 bits.
template <class T>
__device__ __forceinline__ void rotate8(const T *x, int e, bool vec, int half, bool interleaved, int32_t pos,
                                        const float *inv_freq, float (&y)[8]) {
    st::load8(x + e, vec, y);
    if (e >= 2 * half) return;
#pragma unroll 1
    for (int i = 0; i < 8; i++) {
        const int d = e + i;
        if (d >= 2 * half) break;
        const int j = interleaved ? d >> 1 : d < half ? d : d - half;
        const bool second = interleaved ? d & 1 : d >= half;
        const int other = interleaved ? d ^ 1 : second ? d - half : d + half;
        double s, c;
        sincos((double)pos * (double)inv_freq[j], &s, &c);
        const double a = (double)(float)x[d], b = (double)(float)x[other];
        y[i] = (float)(second ? a * c + b * s : a * c - b * s);
    }
}

// Vectors of a token: hq of q, then hkv of k, then hkv of v; LANES lanes each, 8 components a lane.
template <class T, int LANES>
__global__ __launch_bounds__(256) void k_append4(const T *__restrict__ q, const T *__restrict__ k,
                                                 const T *__restrict__ v, T *__restrict__ q_out, T *__restrict__ k_out,
                                                 T *__restrict__ v_out, AppendArgs a) {
    const int per = a.hq + 2 * a.cache.hkv, hkv = a.cache.hkv;
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LANES;
    const int64_t token = i / per;
    const int head = (int)(i - token * per), e = (threadIdx.x % LANES) * 8;
    bool used = token < a.n && e < a.hd;
    int64_t s = 0, pos = 0;
    if (used) {
        s = a.seq[token], pos = a.pos[token];
        used = s >= 0 && s < a.cache.nseq && pos >= 0;
    }
    const int64_t page = used ? page_of(a.cache, s, pos) : -1;
    used = page >= 0;
    float x[8] = {};
    const bool is_q = head < a.hq, is_k = !is_q && head < a.hq + hkv;
    if (used) {
        if (is_q) {
            rotate8(q + token * a.q_stride + (int64_t)head * a.hd, e, a.vec_q, a.half, a.interleaved, (int32_t)pos, a.inv_freq, x);
            st::store8(q_out + (token * a.hq + head) * a.hd + e, a.vec_out, x);
        } else if (is_k) {
            rotate8(k + token * a.k_stride + (int64_t)(head - a.hq) * a.hd, e, a.vec_k, a.half, a.interleaved, (int32_t)pos, a.inv_freq, x);
        } else {
            st::load8(v + token * a.v_stride + (int64_t)(head - a.hq - hkv) * a.hd + e, a.vec_v, x);
        }
    }
    float scale, lo;
    const uint32_t codes = st::quantise8<LANES>(x, used, scale, lo);
    if (!used || is_q) return;
    const int h = head - a.hq - (is_k ? 0 : hkv);
    const int64_t row = (page * hkv + h) * a.cache.page + (pos & (a.cache.page - 1));
    *(uint32_t *)((is_k ? a.k_codes : a.v_codes) + row * (a.hd / 2) + e / 2) = codes;
    if (e == 0) (is_k ? a.k_scales : a.v_scales)[row] = make_float2(scale, lo);
    T *out = is_k ? k_out : v_out;
    if (out) {
        st::values8(codes, scale, lo, x);
        st::store8(out + (token * hkv + h) * a.hd + e, a.vec_out, x);
    }
}

}  // namespace

extern "C" st_status st_kv_append_4bit(const void *q, const void *k, const void *v, int32_t dtype, int64_t n, int64_t hq,
                                       int64_t hkv, int64_t hd, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                       const int32_t *seq, const int32_t *pos, int64_t nseq, const int32_t *table,
                                       int64_t max_pages, int64_t pages, int64_t page, const float *inv_freq, int64_t rot,
                                       int32_t interleaved, uint8_t *k_codes, float *k_scales, uint8_t *v_codes,
                                       float *v_scales, void *q_out, void *k_out, void *v_out, st_stream stream) {
    st::clear_error();
    const char *name = "kv_append_4bit";
    if (!st::heads_ok(name, hq, hkv, hd)) return ST_ERR_INVALID;
    if (n < 0 || n > INT32_MAX) return st::fail(ST_ERR_INVALID, "%s: %lld tokens", name, (long long)n);
    if (dtype < ST_F32 || dtype > ST_BF16) return st::fail(ST_ERR_INVALID, "%s: dtype %d is none of ST_F32, ST_F16, ST_BF16", name, (int)dtype);
    if (rot < 0 || rot > hd || (rot & 1)) return st::fail(ST_ERR_INVALID, "%s: %lld rotated components of %lld (an even number of them)", name, (long long)rot, (long long)hd);
    if ((q && q_stride < hq * hd) || k_stride < hkv * hd || v_stride < hkv * hd)
        return st::fail(ST_ERR_INVALID, "%s: tokens lie %lld, %lld, %lld elements apart, less than their heads", name, (long long)q_stride, (long long)k_stride, (long long)v_stride);
    AppendArgs a = {};
    if (!st::cache_ok(name, a.cache, nseq, table, max_pages, pages, page, hkv, k_codes, k_scales, v_codes, v_scales)) return ST_ERR_INVALID;
    if (n == 0) return ST_OK;
    if (!k || !v || !seq || !pos || (rot && !inv_freq) || (q && !q_out)) return st::fail(ST_ERR_INVALID, "%s: NULL buffer", name);
    const int64_t size = st::dtype_size(dtype);
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)v_out) & (size - 1))
        return st::fail(ST_ERR_INVALID, "%s: a buffer is not aligned to its elements", name);
    if (q && q == q_out) return st::fail(ST_ERR_INVALID, "%s: q_out is q's memory", name);
    if (!st::device_ok()) return ST_ERR_NO_DEVICE;
    const int64_t queries = q ? hq : 0;
    a.n = n, a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride;
    a.hq = (int32_t)queries, a.hd = (int32_t)hd, a.half = (int32_t)rot / 2, a.interleaved = interleaved;
    a.vec_q = st::rows_aligned(q, q_stride, size), a.vec_k = st::rows_aligned(k, k_stride, size), a.vec_v = st::rows_aligned(v, v_stride, size);
    a.vec_out = (((uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0;
    a.seq = seq, a.pos = pos, a.inv_freq = inv_freq;
    a.k_codes = k_codes, a.v_codes = v_codes, a.k_scales = (float2 *)k_scales, a.v_scales = (float2 *)v_scales;
    const int64_t lanes = hd <= 32 ? 4 : hd <= 64 ? 8 : hd <= 128 ? 16 : 32;
    const int64_t blocks = (n * (queries + 2 * hkv) * lanes + 255) / 256;
    if (blocks > INT32_MAX) return st::fail(ST_ERR_INVALID, "%s: %lld tokens of %lld heads are too many for one call", name, (long long)n, (long long)(queries + 2 * hkv));
    return st::with_dtype(dtype, [&](auto *t) -> st_status {
        using T = std::remove_pointer_t<decltype(t)>;
        auto go = [&](auto kernel) {
            kernel<<<(uint32_t)blocks, 256, 0, st::stream_of(stream)>>>((const T *)q, (const T *)k, (const T *)v, (T *)q_out, (T *)k_out,
                                                                        (T *)v_out, a);
        };
        if (lanes == 4)
            go(k_append4<T, 4>);
        else if (lanes == 8)
            go(k_append4<T, 8>);
        else if (lanes == 16)
            go(k_append4<T, 16>);
        else
            go(k_append4<T, 32>);
        ST_LAUNCH_CHECK();
        return ST_OK;
    });
}
