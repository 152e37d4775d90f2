// The paged 4-bit cache as its kernels see it (kv4.hip: append, kv4_attn.hip: attention), and the host's checks of it.
//
// Layout: codes [pages, heads, page, hd / 2] bytes and scales [pages, heads, page] (scale, lo) pairs, for K and for V:
// a head's tokens of a page are contiguous, each one group of the 4-bit format (quant4.h).  Token p of sequence s is in
// page table[s][p / page], slot p % page.
#pragma once

#include "common.h"
#include "quant4.h"

namespace st {

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


inline bool heads_ok(const char *name, int64_t hq, int64_t hkv, int64_t hd) {
    if (hkv < 1 || hq < 1 || hq % hkv || hq > 65535) {
        fail(ST_ERR_INVALID, "%s: %lld query heads over %lld key heads (a multiple, up to 65535)", name, (long long)hq, (long long)hkv);
        return false;
    }
    if (hd != 32 && hd != 64 && hd != 96 && hd != 128 && hd != 192 && hd != 256) {
        fail(ST_ERR_INVALID, "%s: head width %lld is none of 32, 64, 96, 128, 192, 256", name, (long long)hd);
        return false;
    }
    return true;
}

// Checks the cache's sizes and buffers and fills `c`.
inline bool cache_ok(const char *name, Cache &c, int64_t nseq, const int32_t *table, int64_t max_pages, int64_t pages, int64_t page,
              int64_t hkv, const uint8_t *k_codes, const float *k_scales, const uint8_t *v_codes, const float *v_scales) {
    if (nseq < 0 || max_pages < 0 || pages < 0 || pages > INT32_MAX || nseq > 1 << 20) {
        fail(ST_ERR_INVALID, "%s: %lld sequences (up to 2^20) of %lld pages in a cache of %lld (up to 2^31 - 1)", name, (long long)nseq,
                 (long long)max_pages, (long long)pages);
        return false;
    }
    if (page < 16 || page > 1024 || (page & (page - 1))) {
        fail(ST_ERR_INVALID, "%s: pages of %lld tokens are no power of two from 16 to 1024", name, (long long)page);
        return false;
    }
    if (max_pages > (1 << 30) / page) {  // (a tile's keys past the last one stay within 32 bits)
        fail(ST_ERR_INVALID, "%s: %lld pages of %lld tokens a sequence pass 2^30", name, (long long)max_pages, (long long)page);
        return false;
    }
    if (page * hkv * 256 > INT32_MAX) {
        fail(ST_ERR_INVALID, "%s: %lld heads of %lld tokens a page are too many", name, (long long)hkv, (long long)page);
        return false;
    }
    if ((nseq * max_pages > 0 && !table) || (pages > 0 && (!k_codes || !k_scales || !v_codes || !v_scales))) {
        fail(ST_ERR_INVALID, "%s: NULL table or cache", name);
        return false;
    }
    if (((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_scales | (uintptr_t)v_scales) & 15) {
        fail(ST_ERR_INVALID, "%s: the cache's buffers are 16-byte aligned", name);
        return false;
    }
    c = {k_codes, v_codes, (const float2 *)k_scales, (const float2 *)v_scales, table, max_pages, pages, nseq, (int32_t)hkv, (int32_t)page,
         63 - __builtin_clzll((unsigned long long)page)};
    return true;
}

}  // namespace st
