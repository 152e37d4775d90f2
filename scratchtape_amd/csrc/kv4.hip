// The paged 4-bit cache of keys and values: appending new tokens (with the position rotation of queries and keys) and
// causal attention of ragged queries over it.  A token's head vector is one group of the 4-bit format (quant4.h).
//
// Layout: codes [pages, heads, page, hd / 2] bytes and scales [pages, heads, page] (scale, lo) pairs, for K and for V:
// a head's tokens of a page are contiguous.  Token p of sequence s is in page table[s][p / page], slot p % page.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "lanes.h"
#include "quant4.h"

namespace {

struct Cache {
    const uint8_t *k_codes, *v_codes;
    const float2 *k_scales, *v_scales;
    const int32_t *table;
    int64_t max_pages, pages, nseq;
    int32_t hkv, page, page_log2;
};

// The page of token `pos` of sequence `s`, or -1 where the table has none (or one outside the cache).
__device__ __forceinline__ int64_t page_of(const Cache &c, int64_t s, int64_t pos) {
    const int64_t i = pos >> c.page_log2;
    if (i >= c.max_pages) return -1;
    const int64_t p = c.table[s * c.max_pages + i];
    return p >= 0 && p < c.pages ? p : -1;
}

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

// The sequence whose rows q_start[s] .. q_start[s + 1] hold `row` (-1: none).
__device__ __forceinline__ int64_t sequence_of(const int32_t *q_start, int64_t nseq, int64_t row) {
    int64_t lo = 0, hi = nseq;  // the first s with q_start[s + 1] > row
    while (lo < hi) {
        const int64_t mid = (lo + hi) / 2;
        if (q_start[mid + 1] > row)
            hi = mid;
        else
            lo = mid + 1;
    }
    return lo < nseq && q_start[lo] <= row ? lo : -1;
}

// One wave per (row, query head), 64 keys at a time: a lane per key for the scores, then a lane per component.
template <class T>
__global__ __launch_bounds__(64) void k_attention4(const T *__restrict__ q, int64_t n, int32_t hq, int32_t hd,
                                                   int64_t q_stride, const int32_t *__restrict__ q_start,
                                                   const int32_t *__restrict__ kv_len, Cache c, float scale,
                                                   int32_t causal, int64_t window, int32_t one, T *__restrict__ out,
                                                   float *__restrict__ lse) {
    __shared__ float qs[256], ps[64];
    __shared__ int64_t at[64];
    const int lane = threadIdx.x, head = blockIdx.x, h = head / (hq / c.hkv);
    for (int64_t row = blockIdx.y; row < n; row += gridDim.y) {
        const int64_t s = sequence_of(q_start, c.nseq, row);
        if (s < 0) continue;
        const int64_t most = c.max_pages << c.page_log2, len = min((int64_t)max(kv_len[s], 0), most);
        const bool beyond = kv_len[s] > most;  // a length past the table
        const int64_t pos = causal ? len - (q_start[s + 1] - row) : len - 1;
        __syncthreads();
        for (int e = lane; e < hd; e += 64) qs[e] = scale * (float)q[row * q_stride + (int64_t)head * hd + e];
        float m = -INFINITY, l = beyond ? NAN : 0.f, acc[4] = {};
        for (int64_t k0 = window > 0 ? max((int64_t)0, pos - window + 1) / 64 * 64 : 0; k0 <= pos; k0 += 64) {
            const int64_t key = k0 + lane;
            float sc = -INFINITY;
            __syncthreads();
            if (key <= pos && (window <= 0 || key > pos - window)) {
                const int64_t page = page_of(c, s, key);
                const int64_t r = page < 0 ? -1 : (page * c.hkv + h) * c.page + (key & (c.page - 1));
                at[lane] = r;
                if (r >= 0) {
                    float dot = 0.f, sum = 0.f;
                    for (int e = 0; e < hd; e += 8) {
                        const uint32_t w = *(const uint32_t *)(c.k_codes + r * (hd / 2) + e / 2);
                        for (int i = 0; i < 8; i++) {
                            dot += qs[e + i] * (float)((w >> (4 * i)) & 15);
                            sum += qs[e + i];
                        }
                    }
                    const float2 ks = c.k_scales[r];
                    sc = ks.x * dot + ks.y * sum;
                } else {
                    sc = NAN;
                }
            }
            float mt = sc;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) mt = fmaxf(mt, st::xor_lane(mt, o, lane));
            const float mn = fmaxf(m, mt), shift = mn == -INFINITY ? 0.f : mn;
            const float p = sc == -INFINITY ? 0.f : expf(sc - shift), alpha = m == -INFINITY ? 0.f : expf(m - shift);
            float t = p;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) t += st::xor_lane(t, o, lane);
            l = l * alpha + t;
            m = mn;
            ps[lane] = p;
            if (sc == -INFINITY) at[lane] = -1;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int e = lane + 64 * j;
                acc[j] *= alpha;
                if (e >= hd) continue;
                for (int i = 0; i < 64; i++) {
                    const int64_t r = at[i];
                    if (r < 0) continue;
                    const float2 vs = c.v_scales[r];
                    acc[j] += ps[i] * (vs.x * (float)((c.v_codes[r * (hd / 2) + e / 2] >> (4 * (e & 1))) & 15) + vs.y);
                }
            }
        }
        if (one) {  // the phantom logit 0
            const float mn = fmaxf(m, 0.f), alpha = expf(m - mn);
            l = l * alpha + expf(-mn);
            for (int j = 0; j < 4; j++) acc[j] *= alpha;
            m = mn;
        }
        for (int j = 0; j < 4; j++) {
            const int e = lane + 64 * j;
            if (e < hd) out[(row * hq + head) * hd + e] = (T)(l == 0.f ? 0.f : acc[j] / l);
        }
        if (lse && lane == 0) lse[row * hq + head] = l == 0.f ? -INFINITY : m + logf(l);
    }
}

bool heads_ok(const char *name, int64_t hq, int64_t hkv, int64_t hd) {
    if (hkv < 1 || hq < 1 || hq % hkv || hq > 65535) {
        st::fail(ST_ERR_INVALID, "%s: %lld query heads over %lld key heads (a multiple, up to 65535)", name, (long long)hq, (long long)hkv);
        return false;
    }
    if (hd != 32 && hd != 64 && hd != 96 && hd != 128 && hd != 192 && hd != 256) {
        st::fail(ST_ERR_INVALID, "%s: head width %lld is none of 32, 64, 96, 128, 192, 256", name, (long long)hd);
        return false;
    }
    return true;
}

// Checks the cache's sizes and buffers and fills `c`.
bool cache_ok(const char *name, Cache &c, int64_t nseq, const int32_t *table, int64_t max_pages, int64_t pages, int64_t page,
              int64_t hkv, const uint8_t *k_codes, const float *k_scales, const uint8_t *v_codes, const float *v_scales) {
    if (nseq < 0 || max_pages < 0 || pages < 0 || pages > INT32_MAX || nseq > 1 << 20) {
        st::fail(ST_ERR_INVALID, "%s: %lld sequences (up to 2^20) of %lld pages in a cache of %lld (up to 2^31 - 1)", name, (long long)nseq,
                 (long long)max_pages, (long long)pages);
        return false;
    }
    if (page < 16 || page > 1024 || (page & (page - 1))) {
        st::fail(ST_ERR_INVALID, "%s: pages of %lld tokens are no power of two from 16 to 1024", name, (long long)page);
        return false;
    }
    if (max_pages > INT32_MAX / page) {
        st::fail(ST_ERR_INVALID, "%s: %lld pages of %lld tokens a sequence pass 2^31", name, (long long)max_pages, (long long)page);
        return false;
    }
    if ((nseq * max_pages > 0 && !table) || (pages > 0 && (!k_codes || !k_scales || !v_codes || !v_scales))) {
        st::fail(ST_ERR_INVALID, "%s: NULL table or cache", name);
        return false;
    }
    if (((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_scales | (uintptr_t)v_scales) & 15) {
        st::fail(ST_ERR_INVALID, "%s: the cache's buffers are 16-byte aligned", name);
        return false;
    }
    c = {k_codes, v_codes, (const float2 *)k_scales, (const float2 *)v_scales, table, max_pages, pages, nseq, (int32_t)hkv, (int32_t)page,
         63 - __builtin_clzll((unsigned long long)page)};
    return true;
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
    if (!heads_ok(name, hq, hkv, hd)) return ST_ERR_INVALID;
    if (n < 0 || n > INT32_MAX) return st::fail(ST_ERR_INVALID, "%s: %lld tokens", name, (long long)n);
    if (dtype < ST_F32 || dtype > ST_BF16) return st::fail(ST_ERR_INVALID, "%s: dtype %d is none of ST_F32, ST_F16, ST_BF16", name, (int)dtype);
    if (rot < 0 || rot > hd || (rot & 1)) return st::fail(ST_ERR_INVALID, "%s: %lld rotated components of %lld (an even number of them)", name, (long long)rot, (long long)hd);
    if ((q && q_stride < hq * hd) || k_stride < hkv * hd || v_stride < hkv * hd)
        return st::fail(ST_ERR_INVALID, "%s: tokens lie %lld, %lld, %lld elements apart, less than their heads", name, (long long)q_stride, (long long)k_stride, (long long)v_stride);
    AppendArgs a = {};
    if (!cache_ok(name, a.cache, nseq, table, max_pages, pages, page, hkv, k_codes, k_scales, v_codes, v_scales)) return ST_ERR_INVALID;
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

extern "C" int64_t st_kv_attention_4bit_bytes(int64_t n, int64_t nseq, int64_t hq, int64_t hkv, int64_t hd, int64_t max_pages,
                                              int64_t page) {
    return 0;
}

extern "C" st_status st_kv_attention_4bit(const void *q, int32_t dtype, int64_t n, int64_t hq, int64_t hkv, int64_t hd,
                                          int64_t q_stride, const int32_t *q_start, const int32_t *kv_len, int64_t nseq,
                                          const int32_t *table, int64_t max_pages, int64_t pages, int64_t page,
                                          const uint8_t *k_codes, const float *k_scales, const uint8_t *v_codes,
                                          const float *v_scales, float scale, int32_t causal, int64_t window, int32_t one,
                                          void *out, float *lse, void *work, int64_t work_bytes, st_stream stream) {
    st::clear_error();
    const char *name = "kv_attention_4bit";
    if (!heads_ok(name, hq, hkv, hd)) return ST_ERR_INVALID;
    if (n < 0 || n > INT32_MAX) return st::fail(ST_ERR_INVALID, "%s: %lld rows", name, (long long)n);
    if (dtype < ST_F32 || dtype > ST_BF16) return st::fail(ST_ERR_INVALID, "%s: dtype %d is none of ST_F32, ST_F16, ST_BF16", name, (int)dtype);
    if (q_stride < hq * hd) return st::fail(ST_ERR_INVALID, "%s: rows of %lld elements lie %lld apart", name, (long long)(hq * hd), (long long)q_stride);
    if (window < 0 || (window > 0 && !causal)) return st::fail(ST_ERR_INVALID, "%s: a window of %lld keys%s", name, (long long)window, causal ? "" : " without the causal mask");
    Cache c;
    if (!cache_ok(name, c, nseq, table, max_pages, pages, page, hkv, k_codes, k_scales, v_codes, v_scales)) return ST_ERR_INVALID;
    if (n == 0 || nseq == 0) return ST_OK;
    if (!q || !q_start || !kv_len || !out) return st::fail(ST_ERR_INVALID, "%s: NULL buffer", name);
    const int64_t size = st::dtype_size(dtype);
    if (((uintptr_t)q | (uintptr_t)out) & (size - 1)) return st::fail(ST_ERR_INVALID, "%s: q or out not aligned to its elements", name);
    if (!st::device_ok()) return ST_ERR_NO_DEVICE;
    return st::with_dtype(dtype, [&](auto *t) -> st_status {
        using T = std::remove_pointer_t<decltype(t)>;
        k_attention4<T><<<dim3((uint32_t)hq, (uint32_t)std::min<int64_t>(n, 65535)), 64, 0, st::stream_of(stream)>>>(
            (const T *)q, n, (int32_t)hq, (int32_t)hd, q_stride, q_start, kv_len, c, scale, causal, window, one, (T *)out, lse);
        ST_LAUNCH_CHECK();
        return ST_OK;
    });
}
