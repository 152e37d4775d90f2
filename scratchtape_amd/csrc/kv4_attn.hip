// Attention of ragged rows over the paged 4-bit cache (kv4.h).
//
// Row t of sequence s, query head i over key head h, with codes c, scales a and lowest values b of the format, each code
// taken less 8 and b8 = b + 8 a for it (k = aK (cK - 8) + b8K, v = aV (cV - 8) + b8V):
//   z_j = scale (aK_j (q . (cK_j - 8)) + b8K_j sum q)       the score of key j
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(z_j log2 e - M),  M a reference of the row
//   sum_j p_j v_j = sum_j (p_j aV_j) (cV_j - 8) + sum_j p_j b8V_j
// Both products run on the matrix cores (v_mfma_f32_16x16x32_f16), codes as f16 integers from -8 to 7 (exact, a VALU
// operation per code): around 0, so that the rounding of the weights p aV to f16 is not multiplied by an offset.  (Nibbles
// masked in place are f16 subnormals n 2^-24, half the work, and the matrix cores take them; but they line up the sums
// by the exponent that subnormals share, and lose the 6 to 10 bits that n leaves unused: 4e-5 off in f32.)
// Rows are scaled by a power of two to f16 (f32 rows, PARTS = 2, as two f16 parts, 22 bits), scores and sums are f32; the
// weights are rounded to f16, in two parts for f32 rows.
//
// A wave holds 16 RT rows (queries x the heads that share a key head) and takes 32 keys at a time: S^T = K Q^T gives
// each lane 8 scores of one row, which are its B operand of O^T = V^T P^T without a move between lanes.  A row's
// reference M is no running maximum of its scores but follows max(z log2 e + log2 aV), so that p aV stays inside f16's
// normal range whatever the sizes of the values; it is raised only where p aV would pass 2^15, so the common tile has no
// reduction over lanes at all.
// V's operand wants 8 keys of one component in a lane: a lane reads a word (8 components) of 8 keys and v_perm pairs
// their bytes.
//
// A workgroup of 4 waves has a tile of up to 64 RT rows of one sequence and key head, and a chunk of its keys; waves
// without rows of their own share the tile's keys (a single token's rows: all four).  Chunks are cut so that about
// `target` workgroups have equal shares of all sequences' keys together; the lengths are read on the device, and each
// workgroup finds its place by a scan over the sequences.  Where a sequence has several chunks, k_merge4 joins them.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "kv4.h"
#include "lanes.h"
#include "quant4.h"

namespace {

using st::Cache;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int MIN_CHUNK = 256;    // keys: below this a merge costs more than it shares out
constexpr int MAX_CHUNKS = 8192;  // of one sequence (st_kv_attention_4bit keeps target below this)
constexpr float BASE = 7.f, MOST_X = 32768.f;  // p aV is set to 2^7 at most, and may grow to 2^15
constexpr float MIN_E = -86.f, MOST_P = 101.f;  // values below 2^-86 of scale count as that for the reference: p <= 2^93, 2^101

struct AttnArgs {
    Cache c;
    const void *q;
    void *out;
    float *lse;
    const int32_t *q_start, *kv_len;
    float *part_o;    // [part_rows, hd] sums over a chunk's keys
    float2 *part_ml;  // [part_rows] their bounds and totals
    int64_t q_stride, part_rows;
    float scale2;  // scale log2 e
    int32_t n, hq, dtype, causal, window, one, target;
    bool vec_q, vec_out;
};

// A sequence's rows and keys.
struct Seq {
    int first, rows, len, lo, span, tiles;
};

__device__ __forceinline__ Seq seq_of(const AttnArgs &a, int64_t s, int share, int tile_rows, int cap) {
    Seq q;
    const int b = min(max(a.q_start[s], 0), a.n), e = min(max(a.q_start[s + 1], 0), a.n);
    q.first = b;
    q.rows = max(e - b, 0);
    q.len = max(a.kv_len[s], 0);
    // The first key that the first row sees, down to a tile's start.
    const int64_t lo = a.window > 0 ? max((int64_t)0, (int64_t)q.len - q.rows + 1 - a.window) : 0;
    q.lo = (int)(lo & ~31);
    q.span = max(min(q.len, cap) - q.lo, 0);
    q.tiles = (q.rows * share + tile_rows - 1) / tile_rows;
    return q;
}

// Keys per chunk: a multiple of 128, the same in every workgroup (one order of additions).
__device__ __forceinline__ int chunk_keys(const AttnArgs &a, int share, int tile_rows, int cap, int lane) {
    float total = 0.f;
    for (int64_t s0 = 0; s0 < a.c.nseq; s0 += 64) {
        if (s0 + lane < a.c.nseq) {
            const Seq q = seq_of(a, s0 + lane, share, tile_rows, cap);
            total += (float)q.tiles * (float)q.span;
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) total += st::xor_lane(total, o, lane);
    const float each = total * (float)a.c.hkv / (float)a.target;
    const int keys = each < 2.0e9f ? (int)each : 2000000000;
    return max((keys + 127) / 128 * 128, MIN_CHUNK);
}

struct Place {
    Seq q;
    int64_t s;
    int64_t part;  // the first of the sequence's partial rows: row (i hq + head) chunks + chunk
    int chunks, index;
};

// Finds the sequence that has workgroup `w` (by = items) or row `w` (by = rows); false: none has it.
template <bool BY_ITEM>
__device__ __forceinline__ bool place_of(const AttnArgs &a, int64_t w, int share, int tile_rows, int cap, int chunk, int lane,
                                         Place &p) {
    int64_t items = 0, parts = 0;
    for (int64_t s0 = 0; s0 < a.c.nseq; s0 += 64) {
        Seq q = {};
        int mine = 0, chunks = 1;
        if (s0 + lane < a.c.nseq) {
            q = seq_of(a, s0 + lane, share, tile_rows, cap);
            chunks = max((q.span + chunk - 1) / chunk, 1);
            mine = q.tiles * a.c.hkv * chunks;
        }
        // Partial rows of up to 64 sequences in 32 bits: st_kv_attention_4bit bounds their number.
        const int partial = chunks > 1 ? q.rows * a.hq * chunks : 0;
        const int upto = st::wave_incl_scan(mine), parts_upto = st::wave_incl_scan(partial);
        const bool here = BY_ITEM ? items + upto > w : q.first <= w && w < (int64_t)q.first + q.rows;
        const uint64_t any = __ballot(here);
        if (any) {
            const int l = __ffsll((unsigned long long)any) - 1;
            p.s = s0 + l;
            p.q.first = st::lane_value(q.first, l), p.q.rows = st::lane_value(q.rows, l), p.q.len = st::lane_value(q.len, l);
            p.q.lo = st::lane_value(q.lo, l), p.q.span = st::lane_value(q.span, l), p.q.tiles = st::lane_value(q.tiles, l);
            p.chunks = st::lane_value(chunks, l);
            p.part = parts + st::lane_value(parts_upto - partial, l);
            p.index = (int)(w - items) - st::lane_value(upto - mine, l);
            return true;
        }
        items += st::lane_value(upto, 63);
        parts += st::lane_value(parts_upto, 63);
    }
    return false;
}

// The head's components in blocks of 128, 64 or 32: lane column c of a block of width W reads W / 16 components from
// W / 16 c on, which lie in one word.
constexpr int block_width(int hd, int b) {
    return b == 0 ? (hd >= 128 ? 128 : hd >= 64 ? 64 : 32) : hd == 96 ? 32 : hd == 192 ? 64 : hd == 256 ? 128 : 0;
}
constexpr int blocks_of(int hd) { return block_width(hd, 1) ? 2 : 1; }

template <int HD>
struct Tile {
    static constexpr int NW = HD / 32, NB = blocks_of(HD);
    uint32_t k[2][NW];  // of each half of 16 keys: this lane's quarter of one key
    uint32_t v[2][NB][4];
    float4 ks[2][2], vs[2][2];  // (scale, lo) of the lane group's 4 keys
};

template <int NW>
__device__ __forceinline__ void load_words(const uint8_t *p, uint32_t (&w)[NW]) {
    typedef uint32_t v2 __attribute__((ext_vector_type(2)));
    typedef uint32_t v3 __attribute__((ext_vector_type(3), aligned(4)));
    if constexpr (NW % 4 == 0) {
#pragma unroll
        for (int i = 0; i < NW; i += 4) {
            const u4 x = *(const u4 *)(p + 4 * i);
            w[i] = x[0], w[i + 1] = x[1], w[i + 2] = x[2], w[i + 3] = x[3];
        }
    } else if constexpr (NW % 2 == 0) {
#pragma unroll
        for (int i = 0; i < NW; i += 2) {
            const v2 x = *(const v2 *)(p + 4 * i);
            w[i] = x[0], w[i + 1] = x[1];
        }
    } else if constexpr (NW == 3) {
        const v3 x = *(const v3 *)p;
        w[0] = x[0], w[1] = x[1], w[2] = x[2];
    } else {
        w[0] = *(const uint32_t *)p;
    }
}

// Half a tile: 16 keys of page `page`, from slot `slot` on.
template <int HD>
__device__ __forceinline__ void load_half(const Cache &c, int h, int page, int slot, int half, int lane, Tile<HD> &t) {
    const int64_t row = ((int64_t)page * c.hkv + h) * c.page + slot;
    const uint8_t *kb = c.k_codes + row * (HD / 2), *vb = c.v_codes + row * (HD / 2);
    const float4 *ks = (const float4 *)(c.k_scales + row), *vs = (const float4 *)(c.v_scales + row);
    const int col = lane & 15, g = lane >> 4;
    load_words(kb + (col * (HD / 2) + g * (HD / 8)), t.k[half]);
#pragma unroll
    for (int i = 0; i < 2; i++) t.ks[half][i] = ks[2 * g + i], t.vs[half][i] = vs[2 * g + i];
#pragma unroll
    for (int b = 0; b < Tile<HD>::NB; b++) {
        const int width = block_width(HD, b), start = b ? block_width(HD, 0) : 0;
        const int off = start / 2 + 4 * (width == 128 ? col : width == 64 ? col >> 1 : col >> 2);
#pragma unroll
        for (int r = 0; r < 4; r++) t.v[half][b][r] = *(const uint32_t *)(vb + ((4 * g + r) * (HD / 2) + off));
    }
}

__device__ __forceinline__ h8 as_h8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const u4 x = {a, b, c, d};
    return __builtin_bit_cast(h8, x);
}

// Code pairs of a word, less 8: a nibble under f16's exponent of 2^10 reads as 1024 + n (or 1024 + 16 n), which one packed
// f16 operation takes to n - 8 without rounding.  The masks are held in a scalar register and the exponent in a vector
// register that the compiler cannot see through, so that masking and setting the exponent is one v_and_or_b32.
struct Taker {
    uint32_t lower_mask, upper_mask, exponent;

    __device__ __forceinline__ Taker() {
        asm("s_mov_b32 %0, 0x000F000F" : "=s"(lower_mask));
        asm("s_mov_b32 %0, 0x00F000F0" : "=s"(upper_mask));
        asm("v_mov_b32 %0, 0x64006400" : "=v"(exponent));
    }
    __device__ __forceinline__ uint32_t lower(uint32_t x) const {
        const h2 y = __builtin_bit_cast(h2, (x & lower_mask) | exponent) + h2{(_Float16)-1032.f, (_Float16)-1032.f};
        return __builtin_bit_cast(uint32_t, y);
    }
    __device__ __forceinline__ uint32_t upper(uint32_t x) const {
        const h2 y = __builtin_bit_cast(h2, (x & upper_mask) | exponent);
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(y, h2{(_Float16)0.0625f, (_Float16)0.0625f}, h2{(_Float16)-72.f, (_Float16)-72.f}));
    }
    // 8 codes of a word in the order 0 4 1 5 2 6 3 7.
    __device__ __forceinline__ h8 codes8(uint32_t w) const { return as_h8(lower(w), upper(w), lower(w >> 8), upper(w >> 8)); }
};

template <int HD, int PARTS, int RT>
__global__ __launch_bounds__(256, 2) void k_attention4(const AttnArgs a) {
    constexpr int NW = HD / 32, NB = blocks_of(HD), WAVE_ROWS = 16 * RT, TILE_ROWS = 4 * WAVE_ROWS, LDO = HD + 4;
    __shared__ float red[4][WAVE_ROWS][LDO];
    __shared__ float2 ml[4][WAVE_ROWS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const Cache &c = a.c;
    const int share = a.hq / c.hkv, cap = (int)(c.max_pages << c.page_log2);
    const int chunk = chunk_keys(a, share, TILE_ROWS, cap, lane);
    Place pl;
    if (!place_of<true>(a, blockIdx.x, share, TILE_ROWS, cap, chunk, lane, pl)) return;
    // Key heads beside each other (workgroups of one XCD share a head's pages), then the longest tiles first.
    const int h = pl.index % c.hkv, rest = pl.index / c.hkv;
    const int tile = pl.q.tiles - 1 - rest % pl.q.tiles, part = rest / pl.q.tiles;
    if (pl.index < 0 || part >= pl.chunks) return;  // (row starts that do not ascend)
    const int all_rows = pl.q.rows * share, row0 = tile * TILE_ROWS, rows = min(TILE_ROWS, all_rows - row0);
    const int groups = (rows + WAVE_ROWS - 1) / WAVE_ROWS, sharing = groups == 1 ? 4 : groups == 2 ? 2 : 1;
    const int group = wave / sharing, turn = wave % sharing;
    const bool busy = group < groups;

    // This lane's row of each 16, and the positions of the group's first and last.
    int pos[RT];
    const int base = pl.q.len - pl.q.rows;  // position of the first row (negative: more rows than tokens)
    const int first_row = row0 + group * WAVE_ROWS, last_row = min(first_row + WAVE_ROWS, all_rows) - 1;
    const int pos_first = a.causal ? base + first_row / share : pl.q.len - 1;
    const int pos_last = a.causal ? base + last_row / share : pl.q.len - 1;
    h8 qh[RT][NW], ql[PARTS == 2 ? RT : 1][PARTS == 2 ? NW : 1];
    float unscale[RT], qsum[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const int r = first_row + 16 * rt + col;
        pos[rt] = a.causal ? base + min(r, all_rows - 1) / share : pl.q.len - 1;
        float x[NW][8];
        float most = 0.f, sum = 0.f;
        bool finite = true;
        if (busy && r < all_rows) {
            const int64_t at = (int64_t)(pl.q.first + r / share) * a.q_stride + (int64_t)(h * share + r % share) * HD + g * (HD / 4);
#pragma unroll
            for (int w = 0; w < NW; w++) {
                if (a.dtype == ST_F32)
                    st::load8((const float *)a.q + at + 8 * w, a.vec_q, x[w]);
                else if (a.dtype == ST_F16)
                    st::load8((const _Float16 *)a.q + at + 8 * w, a.vec_q, x[w]);
                else
                    st::load8((const __bf16 *)a.q + at + 8 * w, a.vec_q, x[w]);
            }
        } else {
#pragma unroll
            for (int w = 0; w < NW; w++)
#pragma unroll
                for (int i = 0; i < 8; i++) x[w][i] = 0.f;
        }
#pragma unroll
        for (int w = 0; w < NW; w++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                most = fmaxf(most, fabsf(x[w][i]));
                sum += x[w][i];
                finite = finite && __builtin_isfinite(x[w][i]);
            }
        sum = finite ? sum : NAN;  // a row that is not finite: its scores, and so its sums, are NaN
        most = fmaxf(most, st::xor_lane(most, 16, lane));
        most = fmaxf(most, st::xor_lane(most, 32, lane));
        sum += st::xor_lane(sum, 16, lane);
        sum += st::xor_lane(sum, 32, lane);
        // The row's largest component to 2^14 .. 2^15.
        const int e = most > 0.f && __builtin_isfinite(most) ? 15 - __builtin_amdgcn_frexp_expf(most) : 0;
        unscale[rt] = __builtin_amdgcn_ldexpf(a.scale2, -e);
        qsum[rt] = a.scale2 * sum;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            constexpr int order[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float y = __builtin_amdgcn_ldexpf(x[w][order[i]], e);
                qh[rt][w][i] = (_Float16)y;
                if constexpr (PARTS == 2) ql[rt][w][i] = (_Float16)(y - (float)qh[rt][w][i]);
            }
        }
    }

    // The group's keys of this chunk: those that its first row may see up to those of its last, within the table.
    int begin = pl.q.lo + part * chunk, end = (int)min(min((int64_t)begin + chunk, (int64_t)pos_last + 1), (int64_t)cap);
    if (a.window > 0) begin = max(begin, (int)(max((int64_t)0, (int64_t)pos_first + 1 - a.window) & ~31));
    const int first_key = begin + 32 * turn, step = 32 * sharing;
    const int count = busy && c.pages > 0 && end > first_key ? (end - first_key + step - 1) / step : 0;
    const bool no_pages = busy && c.pages == 0 && end > begin;

    f4 o[RT][HD / 16];
    float ref[RT], total[RT], low[RT];  // sums in units of 2^ref
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        ref[rt] = -INFINITY, total[rt] = low[rt] = 0.f;
#pragma unroll
        for (int j = 0; j < HD / 16; j++) o[rt][j] = f4{0.f, 0.f, 0.f, 0.f};
    }
    uint32_t sel[NB][4];
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int width = block_width(HD, b), byte = width == 128 ? i : width == 64 ? 2 * (col & 1) + (i & 1) : col & 3;
            sel[b][i] = 0x0c000c00u | (uint32_t)(4 + byte) << 16 | (uint32_t)byte;
        }

    const Taker take;
    // Pages of the next 32 tiles' halves, a half a lane: -1 one outside the cache, 0 (not looked at) behind the end.
    int entries = 0, entries_to = 0;
    auto load_entries = [&](int it) {
        const int key = first_key + (it + (lane >> 1)) * step + 16 * (lane & 1);
        entries = 0;
        if (key < end) {
            const int p = c.table[pl.s * c.max_pages + (key >> c.page_log2)];
            entries = p >= 0 && p < c.pages ? p : -1;
        }
    };
    auto load_tile = [&](int it, Tile<HD> &t, int &bad) {
        if (it >= entries_to) load_entries(it), entries_to = it + 32;
        const int key = first_key + it * step;
        const int at = 2 * (it + 32 - entries_to), p0 = st::lane_value(entries, at), p1 = st::lane_value(entries, at + 1);
        bad = (p0 < 0 ? 1 : 0) | (p1 < 0 ? 2 : 0);
        load_half<HD>(c, h, max(p0, 0), key & (c.page - 1), 0, lane, t);
        load_half<HD>(c, h, max(p1, 0), (key + 16) & (c.page - 1), 1, lane, t);
    };

    auto scores = [&](auto masked_, const f4 (&s)[RT][2], const float (&ak)[2][4], const float (&bk)[2][4], int key0, int rt,
                      float shift, float (&z)[2][4]) {
        constexpr bool masked = decltype(masked_)::value;
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                z[i][r] = __builtin_fmaf(ak[i][r], s[rt][i][r] * unscale[rt], __builtin_fmaf(bk[i][r], qsum[rt], shift));
                if constexpr (masked) {
                    const int key = key0 + 16 * i + r;
                    const bool seen = key <= pos[rt] && (a.window <= 0 || key > pos[rt] - a.window);
                    z[i][r] = seen ? z[i][r] : -INFINITY;
                }
            }
    };

    auto work_on = [&](auto masked_, const Tile<HD> &t, int kt, int bad) {
        constexpr bool masked = decltype(masked_)::value;
        const int key0 = kt + 4 * g;
        f4 s[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) s[rt][0] = s[rt][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const h8 k8 = take.codes8(t.k[i][w]);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    s[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, qh[rt][w], s[rt][i], 0, 0, 0);
                    if constexpr (PARTS == 2) s[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, ql[rt][w], s[rt][i], 0, 0, 0);
                }
            }
        float ak[2][4], bk[2][4], av[2][4], bv[2][4];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float4 x = t.ks[i][r >> 1], y = t.vs[i][r >> 1];
                ak[i][r] = r & 1 ? x.z : x.x, bk[i][r] = r & 1 ? x.w : x.y;
                av[i][r] = r & 1 ? y.z : y.x, bv[i][r] = r & 1 ? y.w : y.y;
            }
        if (bad) {  // keys on a page outside the cache: NaN to the rows that see them
#pragma unroll
            for (int r = 0; r < 4; r++) {
                if (bad & 1) ak[0][r] = NAN, av[0][r] = 0.f, bv[0][r] = 0.f;
                if (bad & 2) ak[1][r] = NAN, av[1][r] = 0.f, bv[1][r] = 0.f;
            }
        }
        if constexpr (masked) {  // what lies behind the end never counts, whatever it holds
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (key0 + 16 * i + r >= end) av[i][r] = bv[i][r] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 2; i++)  // what a code of 8 stands for
#pragma unroll
            for (int r = 0; r < 4; r++) bk[i][r] = __builtin_fmaf(8.f, ak[i][r], bk[i][r]), bv[i][r] = __builtin_fmaf(8.f, av[i][r], bv[i][r]);
        // p = 2^(z - R) and p aV of every row; R is raised where p aV would pass f16's range or p an f32's.
        float p[RT][2][4], x[RT][2][4];
        float most_z = -INFINITY, most_x = 0.f;
        auto weigh = [&](int rt) {
            scores(masked_, s, ak, bk, key0, rt, -ref[rt], p[rt]);
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    most_z = fmaxf(most_z, p[rt][i][r]);
                    p[rt][i][r] = __builtin_amdgcn_exp2f(p[rt][i][r]);
                    x[rt][i][r] = p[rt][i][r] * av[i][r];
                    if (masked && p[rt][i][r] == 0.f) x[rt][i][r] = 0.f;  // not 0 times a NaN
                    most_x = fmaxf(most_x, x[rt][i][r]);
                }
        };
#pragma unroll
        for (int rt = 0; rt < RT; rt++) weigh(rt);
        if (__any(most_z > MOST_P || most_x > MOST_X)) {
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                float z[2][4];
                scores(masked_, s, ak, bk, key0, rt, 0.f, z);
                float m = -INFINITY;
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float e = av[i][r] > 0.f ? (float)__builtin_amdgcn_frexp_expf(av[i][r]) : MIN_E;
                        m = fmaxf(m, z[i][r] + fmaxf(e, MIN_E));
                    }
                m = fmaxf(m, st::xor_lane(m, 16, lane));
                m = fmaxf(m, st::xor_lane(m, 32, lane));
                m = fmaxf(ref[rt], m - BASE);
                const float keep = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ref[rt] - m);
                total[rt] *= keep, low[rt] *= keep;
#pragma unroll
                for (int j = 0; j < HD / 16; j++) o[rt][j] *= keep;
                ref[rt] = m;
                weigh(rt);
            }
        }
        h8 ph[RT], pr[PARTS == 2 ? RT : 1];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    total[rt] += p[rt][i][r];
                    float y = p[rt][i][r] * bv[i][r];
                    if (masked && p[rt][i][r] == 0.f) y = 0.f;
                    low[rt] += y;
                    ph[rt][4 * i + r] = (_Float16)x[rt][i][r];
                    if constexpr (PARTS == 2) pr[rt][4 * i + r] = (_Float16)(x[rt][i][r] - (float)ph[rt][4 * i + r]);
                }
        }
#pragma unroll
        for (int b = 0; b < NB; b++) {
            constexpr int first = block_width(HD, 0) / 16;
            const int bytes = block_width(HD, b) / 32;
#pragma unroll
            for (int i = 0; i < bytes; i++) {
                const uint32_t x0 = __builtin_amdgcn_perm(t.v[0][b][1], t.v[0][b][0], sel[b][i]);
                const uint32_t x1 = __builtin_amdgcn_perm(t.v[0][b][3], t.v[0][b][2], sel[b][i]);
                const uint32_t x2 = __builtin_amdgcn_perm(t.v[1][b][1], t.v[1][b][0], sel[b][i]);
                const uint32_t x3 = __builtin_amdgcn_perm(t.v[1][b][3], t.v[1][b][2], sel[b][i]);
                const h8 even = as_h8(take.lower(x0), take.lower(x1), take.lower(x2), take.lower(x3));
                const h8 odd = as_h8(take.upper(x0), take.upper(x1), take.upper(x2), take.upper(x3));
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    f4 &e = o[rt][b * first + 2 * i], &d = o[rt][b * first + 2 * i + 1];
                    e = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, ph[rt], e, 0, 0, 0);
                    d = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, ph[rt], d, 0, 0, 0);
                    if constexpr (PARTS == 2) {
                        e = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, pr[rt], e, 0, 0, 0);
                        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, pr[rt], d, 0, 0, 0);
                    }
                }
            }
        }
    };

    auto process = [&](const Tile<HD> &t, int it, int bad) {
        const int kt = first_key + it * step;
        if (kt + 31 > pos_first || kt + 31 >= end || (a.window > 0 && kt <= pos_last - a.window))
            work_on(std::true_type(), t, kt, bad);
        else
            work_on(std::false_type(), t, kt, bad);
    };

    if (count > 0) {
        // The next tile's loads are in flight while one is worked on.  They are issued without a condition (the last tile again
        // behind the end): the wait for a tile would else have to be one for everything.
        Tile<HD> t0, t1;
        int bad0, bad1;
        load_tile(0, t0, bad0);
        for (int it = 0; it < count; it += 2) {
            load_tile(min(it + 1, count - 1), t1, bad1);
            process(t0, it, bad0);
            load_tile(min(it + 2, count - 1), t0, bad0);
            if (it + 1 < count) process(t1, it + 1, bad1);
        }
    }

    // Each wave's sums in true units against its own bound, then against the bound of the waves that share its rows.
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        total[rt] += st::xor_lane(total[rt], 16, lane);
        total[rt] += st::xor_lane(total[rt], 32, lane);
        low[rt] += st::xor_lane(low[rt], 16, lane);
        low[rt] += st::xor_lane(low[rt], 32, lane);
        // A row whose own token lies past the table (or that sees a token of a cache without pages).
        if (pos[rt] >= cap || no_pages) total[rt] = NAN;
        if (g == 0) ml[wave][16 * rt + col] = make_float2(ref[rt], total[rt]);
    }
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        float m = -INFINITY;
        for (int i = 0; i < sharing; i++) m = fmaxf(m, ml[group * sharing + i][16 * rt + col].x);
        const float factor = ref[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref[rt] - m);
        const float off = low[rt] * factor;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            constexpr int first = block_width(HD, 0) / 16;
            const int per = block_width(HD, b) / 16, start = b ? block_width(HD, 0) : 0;
#pragma unroll
            for (int j = 0; j < per; j++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    red[wave][16 * rt + col][start + per * (4 * g + r) + j] = __builtin_fmaf(o[rt][b * first + j][r], factor, off);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * (HD / 8); i += 256) {
        const int x = i / (HD / 8), e = 8 * (i % (HD / 8)), w0 = x / WAVE_ROWS * sharing, y = x % WAVE_ROWS;
        float m = -INFINITY, l = 0.f, v[8] = {};
        for (int k = 0; k < sharing; k++) m = fmaxf(m, ml[w0 + k][y].x);
        for (int k = 0; k < sharing; k++) {
            const float2 t = ml[w0 + k][y];
            l += t.y * (t.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(t.x - m));
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] += red[w0 + k][y][e + j];
        }
        const int r = row0 + x, head = h * share + r % share;
        const int64_t row = ((int64_t)pl.q.first + r / share) * a.hq + head;
        if (pl.chunks > 1) {
            const int64_t slot = pl.part + ((int64_t)(r / share) * a.hq + head) * pl.chunks + part;
            if (slot < 0 || slot >= a.part_rows) continue;
            st::store8(a.part_o + slot * HD + e, true, v);
            if (e == 0) a.part_ml[slot] = make_float2(m, l);
            continue;
        }
        const float top = a.one ? fmaxf(m, 0.f) : m, f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
        const float sum = l * f + (a.one ? __builtin_amdgcn_exp2f(-top) : 0.f), inv = sum == 0.f ? 0.f : f / sum;
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] *= inv;
        if (a.dtype == ST_F32)
            st::store8((float *)a.out + row * HD + e, a.vec_out, v);
        else if (a.dtype == ST_F16)
            st::store8((_Float16 *)a.out + row * HD + e, a.vec_out, v);
        else
            st::store8((__bf16 *)a.out + row * HD + e, a.vec_out, v);
        if (a.lse && e == 0) a.lse[row] = sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * 0.693147180559945309f;
    }
}

// Joins the chunks of the rows whose sequences have several: out = sum_c 2^(M_c - M) O_c / sum_c 2^(M_c - M) l_c.
template <int HD>
__global__ __launch_bounds__(256) void k_merge4(const AttnArgs a, int tile_rows) {
    constexpr int LANES = HD / 4, GROUPS = 256 / LANES;
    __shared__ float weight[MAX_CHUNKS];
    __shared__ float red[GROUPS][HD], stat[8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Cache &c = a.c;
    const int share = a.hq / c.hkv, cap = (int)(c.max_pages << c.page_log2);
    const int chunk = chunk_keys(a, share, tile_rows, cap, lane);
    const int64_t pairs = (int64_t)a.n * a.hq;
    for (int64_t pair = blockIdx.x; pair < pairs; pair += gridDim.x) {
        const int row = (int)(pair / a.hq), head = (int)(pair - (int64_t)row * a.hq);
        Place pl;
        if (!place_of<false>(a, row, share, tile_rows, cap, chunk, lane, pl) || pl.chunks == 1 || pl.chunks > MAX_CHUNKS) continue;
        const int64_t slot = pl.part + ((int64_t)(row - pl.q.first) * a.hq + head) * pl.chunks;
        if (slot < 0 || slot + pl.chunks > a.part_rows) continue;
        float m = -INFINITY, l = 0.f;
        for (int i = threadIdx.x; i < pl.chunks; i += 256) m = fmaxf(m, a.part_ml[slot + i].x);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, st::xor_lane(m, o, lane));
        __syncthreads();  // the last pair's readers are done
        if (lane == 0) stat[wave] = m;
        __syncthreads();
        m = fmaxf(fmaxf(stat[0], stat[1]), fmaxf(stat[2], stat[3]));
        for (int i = threadIdx.x; i < pl.chunks; i += 256) {
            const float2 t = a.part_ml[slot + i];
            const float w = t.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(t.x - m);
            weight[i] = w;
            l += t.y * w;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) l += st::xor_lane(l, o, lane);
        if (lane == 0) stat[4 + wave] = l;
        __syncthreads();
        l = (stat[4] + stat[5]) + (stat[6] + stat[7]);
        const int gr = threadIdx.x / LANES, e = 4 * (threadIdx.x % LANES);
        if (gr < GROUPS) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int i = gr; i < pl.chunks; i += GROUPS) {
                const float w = weight[i];
                const float4 x = *(const float4 *)(a.part_o + (slot + i) * HD + e);
                v.x += w * x.x, v.y += w * x.y, v.z += w * x.z, v.w += w * x.w;
            }
            *(float4 *)&red[gr][e] = v;
        }
        __syncthreads();
        const float top = a.one ? fmaxf(m, 0.f) : m, f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
        const float sum = l * f + (a.one ? __builtin_amdgcn_exp2f(-top) : 0.f), inv = sum == 0.f ? 0.f : f / sum;
        if ((int)threadIdx.x < HD) {
            float v = 0.f;
#pragma unroll
            for (int i = 0; i < GROUPS; i++) v += red[i][threadIdx.x];
            v *= inv;
            const int64_t at = pair * HD + threadIdx.x;
            if (a.dtype == ST_F32)
                ((float *)a.out)[at] = v;
            else if (a.dtype == ST_F16)
                ((_Float16 *)a.out)[at] = (_Float16)v;
            else
                ((__bf16 *)a.out)[at] = (__bf16)v;
        }
        if (a.lse && threadIdx.x == 0) a.lse[pair] = sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * 0.693147180559945309f;
    }
}

// How a call is cut: rows per wave, workgroups to aim at, and the partial rows that it can need.
struct Cut {
    int rt, target;
    int64_t part_rows;
};

Cut cut_of(int64_t n, int64_t nseq, int64_t hq, int64_t hkv, int64_t hd, int64_t max_pages, int64_t page) {
    Cut c;
    // Sequences of many rows: 32 rows a wave, which share the work of taking codes apart.
    c.rt = hd <= 128 && n * (hq / hkv) >= 64 * nseq ? 2 : 1;
    c.target = 4 * st::device_cus();
    const int64_t keys = max_pages * page, tile = 64 * c.rt;
    const int64_t chunks = std::min<int64_t>((keys + MIN_CHUNK - 1) / MIN_CHUNK, c.target + 2);
    // A sequence of `chunks` > 1 chunks has at most twice as many as its share of the target.
    c.part_rows = keys <= MIN_CHUNK ? 0 : std::min<int64_t>(n * hq * chunks, (int64_t)2 * c.target * tile + tile);
    return c;
}

}  // namespace

extern "C" int64_t st_kv_attention_4bit_bytes(int64_t n, int64_t nseq, int64_t hq, int64_t hkv, int64_t hd, int64_t max_pages,
                                              int64_t page) {
    if (n <= 0 || nseq <= 0 || hkv <= 0 || hq < hkv || max_pages <= 0) return 0;
    return cut_of(n, nseq, hq, hkv, hd, max_pages, page).part_rows * (hd + 2) * 4;
}

extern "C" st_status st_kv_attention_4bit(const void *q, int32_t dtype, int64_t n, int64_t hq, int64_t hkv, int64_t hd,
                                          int64_t q_stride, const int32_t *q_start, const int32_t *kv_len, int64_t nseq,
                                          const int32_t *table, int64_t max_pages, int64_t pages, int64_t page,
                                          const uint8_t *k_codes, const float *k_scales, const uint8_t *v_codes,
                                          const float *v_scales, float scale, int32_t causal, int64_t window, int32_t one,
                                          void *out, float *lse, void *work, int64_t work_bytes, st_stream stream) {
    st::clear_error();
    const char *name = "kv_attention_4bit";
    if (!st::heads_ok(name, hq, hkv, hd)) return ST_ERR_INVALID;
    if (n < 0 || n > INT32_MAX / hq / 256) return st::fail(ST_ERR_INVALID, "%s: %lld rows of %lld heads (up to 2^23 in all)", name, (long long)n, (long long)hq);
    if (dtype < ST_F32 || dtype > ST_BF16) return st::fail(ST_ERR_INVALID, "%s: dtype %d is none of ST_F32, ST_F16, ST_BF16", name, (int)dtype);
    if (q_stride < hq * hd) return st::fail(ST_ERR_INVALID, "%s: rows of %lld elements lie %lld apart", name, (long long)(hq * hd), (long long)q_stride);
    if (window < 0 || (window > 0 && !causal)) return st::fail(ST_ERR_INVALID, "%s: a window of %lld keys%s", name, (long long)window, causal ? "" : " without the causal mask");
    AttnArgs a = {};
    if (!st::cache_ok(name, a.c, nseq, table, max_pages, pages, page, hkv, k_codes, k_scales, v_codes, v_scales)) return ST_ERR_INVALID;
    if (n == 0 || nseq == 0) return ST_OK;
    if (!q || !q_start || !kv_len || !out) return st::fail(ST_ERR_INVALID, "%s: NULL buffer", name);
    const int64_t size = st::dtype_size(dtype);
    if (((uintptr_t)q | (uintptr_t)out) & (size - 1)) return st::fail(ST_ERR_INVALID, "%s: q or out not aligned to its elements", name);
    const Cut cut = cut_of(n, nseq, hq, hkv, hd, max_pages, page);
    if (cut.part_rows > 0 && (!work || ((uintptr_t)work & 15) || work_bytes < cut.part_rows * (hd + 2) * 4))
        return st::fail(ST_ERR_INVALID, "%s: work is %lld bytes of 16-byte aligned device memory, got %lld", name,
                        (long long)(cut.part_rows * (hd + 2) * 4), (long long)(work ? work_bytes : 0));
    if (!st::device_ok()) return ST_ERR_NO_DEVICE;
    a.q = q, a.out = out, a.lse = lse, a.q_start = q_start, a.kv_len = kv_len;
    a.part_o = (float *)work, a.part_ml = (float2 *)((float *)work + cut.part_rows * hd), a.part_rows = cut.part_rows;
    a.q_stride = q_stride;
    a.scale2 = scale * 1.44269504088896341f;
    a.n = (int32_t)n, a.hq = (int32_t)hq, a.dtype = dtype, a.causal = causal != 0, a.one = one != 0;
    a.window = window > INT32_MAX / 2 ? 0 : (int32_t)window;
    a.target = cut.target;
    a.vec_q = st::rows_aligned(q, q_stride, size), a.vec_out = ((uintptr_t)out & 15) == 0;
    const int64_t tile = 64 * cut.rt, share = hq / hkv;
    // Every tile once, and the target's worth of further chunks (a little more for the rounding of the f32 total).
    const int64_t grid = hkv * (n * share / tile + nseq) + (cut.part_rows > 0 ? cut.target + cut.target / 64 + 64 : 0);
    if (grid > INT32_MAX) return st::fail(ST_ERR_INVALID, "%s: %lld rows and %lld sequences are too many for one call", name, (long long)n, (long long)nseq);
    auto go = [&](auto hd_) -> st_status {
        constexpr int HD = decltype(hd_)::value;
        const hipStream_t s = st::stream_of(stream);
        if (cut.rt == 1) {
            if (dtype == ST_F32)
                k_attention4<HD, 2, 1><<<(uint32_t)grid, 256, 0, s>>>(a);
            else
                k_attention4<HD, 1, 1><<<(uint32_t)grid, 256, 0, s>>>(a);
        } else if constexpr (HD <= 128) {
            if (dtype == ST_F32)
                k_attention4<HD, 2, 2><<<(uint32_t)grid, 256, 0, s>>>(a);
            else
                k_attention4<HD, 1, 2><<<(uint32_t)grid, 256, 0, s>>>(a);
        }
        ST_LAUNCH_CHECK();
        if (cut.part_rows > 0) {
            k_merge4<HD><<<(uint32_t)std::min<int64_t>(n * hq, 8 * st::device_cus()), 256, 0, s>>>(a, (int)tile);
            ST_LAUNCH_CHECK();
        }
        return ST_OK;
    };
    switch (hd) {
        case 32:
            return go(std::integral_constant<int, 32>());
        case 64:
            return go(std::integral_constant<int, 64>());
        case 96:
            return go(std::integral_constant<int, 96>());
        case 128:
            return go(std::integral_constant<int, 128>());
        case 192:
            return go(std::integral_constant<int, 192>());
        default:
            return go(std::integral_constant<int, 256>());
    }
}
