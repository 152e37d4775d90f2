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
    int32_t hq, hd, half, interleaved, stretch;
    bool vec, vec_out;
    const int32_t *seq, *pos;
    const float *inv_freq;
    uint8_t *k_codes, *v_codes;
    float2 *k_scales, *v_scales;
    Cache cache;
};

// A lane's part of the rotation: component e + i becomes x[i] c[i] + other[i] s[i], `other` the second of its pair.
struct Turn {
    double c[8], s[8];
    __device__ __forceinline__ Turn(const double2 *turn, int e, int half, bool interleaved) {  // turn: (cos, sin) of the pairs' angles
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int d = e + i;
            const bool second = interleaved ? d & 1 : d >= half;
            const double2 t = turn[d >= 2 * half ? 0 : interleaved ? d >> 1 : second ? d - half : d];
            c[i] = t.x, s[i] = second ? t.y : -t.y;
        }
    }
    __device__ __forceinline__ void operator()(int e, int half, float (&x)[8], const float (&other)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (e + i < 2 * half) x[i] = (float)((double)x[i] * c[i] + (double)other[i] * s[i]);
    }
};

// Eight elements as they lie in memory.  vec: they are 16-byte aligned.
template <class T>
struct Eight {
    typedef T V __attribute__((ext_vector_type(8), aligned(16)));
    V v;
    __device__ __forceinline__ void load(const T *p, bool vec) {
        if (vec) {
            v = *(const V *)p;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = p[i];
        }
    }
};

// A token's vectors (hq of q, then hkv of k, then hkv of v), `stretch` of them a workgroup, LANES lanes each, 8 components a
// lane.  The cosines and sines are taken once a workgroup, in 64 bits; sequence, position and page are the same for all its
// lanes. 8191 tokens of 48 vectors of 128 in f16, 210 MB: 58 us (3.6 TB/s; 68 with loads behind the page's and the angles' and
// five waves a SIMD instead of six, for which some registers are put away around the sines; 233 with the angles taken for each
// component and 64-bit quotients).  Bound by waits for loads.  In f32, 420 MB, 202 us (2.1 TB/s): 18 registers are put away there, 10 in
// the 16-bit types.
template <class T, int LANES>
__global__ __launch_bounds__(256, 6) void k_append4(const T *__restrict__ q, const T *__restrict__ k,
                                                 const T *__restrict__ v, T *__restrict__ q_out, T *__restrict__ k_out,
                                                 T *__restrict__ v_out, AppendArgs a) {
    __shared__ double2 turn[128];
    const int hq = a.hq, hkv = a.cache.hkv, e = (threadIdx.x % LANES) * 8;
    const int64_t token = (int64_t)blockIdx.z * gridDim.x + blockIdx.x;
    if (token >= a.n) return;
    const int begin = blockIdx.y * a.stretch, end = min(begin + a.stretch, hq + 2 * hkv);
    // The lane's components of a vector and the seconds of their pairs, a pass ahead (lanes without a vector repeat another's).
    Eight<T> mine, pairs;
    const int es = e < a.hd ? e : 0;
    auto fetch = [&](int first) {
        const int head = min(first + (int)threadIdx.x / LANES, end - 1);
        const bool is_q = head < hq, is_k = !is_q && head < hq + hkv;
        const T *from = is_q ? q + token * a.q_stride + (int64_t)head * a.hd
                             : is_k ? k + token * a.k_stride + (int64_t)(head - hq) * a.hd : v + token * a.v_stride + (int64_t)(head - hq - hkv) * a.hd;
        mine.load(from + es, a.vec);
        if (a.interleaved) return;
        if (a.half % 8 == 0) {  // the eight others lie side by side
            pairs.load(from + (es >= 2 * a.half ? es : es >= a.half ? es - a.half : es + a.half), a.vec);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) pairs.v[i] = from[es + i >= 2 * a.half ? es + i : es + i >= a.half ? es + i - a.half : es + i + a.half];
        }
    };
    fetch(begin);
    const int64_t s = a.seq[token], pos = a.pos[token];
    if (s < 0 || s >= a.cache.nseq || pos < 0) return;
    const int64_t page = page_of(a.cache, s, pos);
    if (page < 0) return;
    if (a.half && begin < hq + hkv) {
        if ((int)threadIdx.x < a.half) {
            double si, co;
            sincos((double)pos * (double)a.inv_freq[threadIdx.x], &si, &co);
            turn[threadIdx.x] = make_double2(co, si);
        }
        __syncthreads();
    }
    const Turn rotate(turn, e, a.half, a.interleaved);
    for (int first = begin; first < end; first += 256 / LANES) {
        const int head = first + threadIdx.x / LANES;
        const bool used = head < end && e < a.hd, is_q = head < hq, is_k = !is_q && head < hq + hkv;
        const int h = is_q ? head : is_k ? head - hq : head - hq - hkv;
        float x[8], other[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (float)mine.v[i], other[i] = (float)(a.interleaved ? mine.v[i ^ 1] : pairs.v[i]);
        if (first + 256 / LANES < end) fetch(first + 256 / LANES);
        if (head < hq + hkv) rotate(e, a.half, x, other);
        if (used && is_q) st::store8(q_out + (token * hq + h) * a.hd + e, a.vec_out, x);
        if (first + 256 / LANES <= hq) continue;  // queries only
        float scale, lo;
        const uint32_t codes = st::quantise8<LANES>(x, used, scale, lo);
        if (!used || is_q) continue;
        const int64_t row = (page * hkv + h) * a.cache.page + (pos & (a.cache.page - 1));
        *(uint32_t *)((is_k ? a.k_codes : a.v_codes) + row * (a.hd / 2) + e / 2) = codes;
        if (e == 0) (is_k ? a.k_scales : a.v_scales)[row] = make_float2(scale, lo);
        T *out = is_k ? k_out : v_out;
        if (out) {
            st::values8(codes, scale, lo, x);
            st::store8(out + (token * hkv + h) * a.hd + e, a.vec_out, x);
        }
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
    if (dtype < ST_F32 || dtype > ST_BF16)
        return st::fail(ST_ERR_INVALID, "%s: dtype %d is none of ST_F32, ST_F16, ST_BF16",
                        name, (int)dtype);
    if (rot < 0 || rot > hd || (rot & 1))
        return st::fail(ST_ERR_INVALID, "%s: %lld rotated components of %lld (an even number of them)",
                        name, (long long)rot, (long long)hd);
    if ((q && q_stride < hq * hd) || k_stride < hkv * hd || v_stride < hkv * hd)
        return st::fail(ST_ERR_INVALID, "%s: tokens lie %lld, %lld, %lld elements apart, less than their heads",
                        name, (long long)q_stride, (long long)k_stride, (long long)v_stride);
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
    a.vec = (!q || st::rows_aligned(q, q_stride, size)) && st::rows_aligned(k, k_stride, size) && st::rows_aligned(v, v_stride, size);
    a.vec_out = (((uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0;
    a.seq = seq, a.pos = pos, a.inv_freq = inv_freq;
    a.k_codes = k_codes, a.v_codes = v_codes, a.k_scales = (float2 *)k_scales, a.v_scales = (float2 *)v_scales;
    const int64_t lanes = hd <= 32 ? 4 : hd <= 64 ? 8 : hd <= 128 ? 16 : 32;
    // With a token for every CU a workgroup takes a whole token, and its sines once; with fewer, one pass of its vectors.  us, whole
    // and one pass, bf16 of 48 vectors of 128: 64 tokens 7.0 and 6.1, 256 7.8 and 8.0, 512 9.9 and 11.1, 1024 13.1 and 16.8, 8191 64
    // and 98; f32: 64 9.3 and 7.2, 128 9.7 and 9.4, 256 11.7 and 12.7, 8191 202 and 220; f16 of 21 vectors of 96: 128 6.8 and 6.3,
    // 256 7.2 and 7.1, 512 8.5 and 9.0; of 20 of 256: 128 7.3 and 7.0, 256 7.7 and 8.3.
    const int64_t vectors = queries + 2 * hkv, once = 256 / lanes;
    a.stretch = (int32_t)(n >= st::device_cus() ? vectors : once);
    const int64_t along = std::min<int64_t>(n, 1 << 23);  // (a launch holds less than 2^32 threads along x)
    const dim3 grid((uint32_t)along, (uint32_t)((vectors + a.stretch - 1) / a.stretch), (uint32_t)((n + along - 1) / along));
    return st::with_dtype(dtype, [&](auto *t) -> st_status {
        using T = std::remove_pointer_t<decltype(t)>;
        auto go = [&](auto kernel) {
            kernel<<<grid, 256, 0, st::stream_of(stream)>>>((const T *)q, (const T *)k, (const T *)v, (T *)q_out, (T *)k_out,
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
