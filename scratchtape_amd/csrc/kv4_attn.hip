// Attention of ragged rows over the paged 4-bit cache (kv4.h).
//
// Row t of sequence s, query head i over key head h, with codes c, scales a and lowest values b of the format, each code
// taken less 8 and b8 = b + 8 a for it (k = aK (cK - 8) + b8K, v = aV (cV - 8) + b8V):
//   z_j = scale (aK_j (q . (cK_j - 8)) + b8K_j sum q)       the score of key j
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(z_j log2 e - M),  M a reference of the row
//   sum_j p_j v_j = sum_j (p_j aV_j) (cV_j - 8) + sum_j p_j b8V_j
// Both products run on the matrix cores, codes as f16 integers from -8 to 7 (exact, a VALU operation per code): around 0, so
// that the rounding of the weights p aV to f16 is not multiplied by an offset.  (Nibbles masked in place are f16 subnormals n
// 2^-24, half the work, and the matrix cores take them; but they line up the sums by the exponent that subnormals share, and
// lose the 6 to 10 bits that n leaves unused: 4e-5 off in f32.) Rows are scaled by a power of two to f16 (f32 rows, PARTS = 2,
// as two f16 parts, 22 bits), scores and sums are f32; the weights are rounded to f16, in two parts for f32 rows and for few
// rows of f16.  A row's reference M is no running maximum of its scores but follows max(z log2 e + log2 aV), so that p aV stays
// inside f16's normal range whatever the sizes of the values (and where |b8| is far above aV, as in a vector of equal components,
// follows that, so that p b8 stays inside f32's); it is raised only where p aV would pass 2^15, p or p b8 a bound of theirs, so
// the common tile has no reduction over lanes at all.
//
// What the kernel spends is the taking apart of codes, about a VALU operation each for K and for V, and the scores'
// arithmetic; both would leave memory waiting, so the rest is arranged around them.  A wave has 16 RT rows and takes 32 keys at
// a time.  S^T = K Q^T (16x16x32) gives a lane 8 scores of one row, which are its B operand of O^T = V^T P^T without a move
// between lanes.  (Few rows leave columns empty.  A kernel for up to 8 of them with a key a lane, 4x4x4 products, took
// 83 and 43 us where this one takes 86 and 45, 64 sequences and one long one, but 27 and 113 where this takes 21 and 89,
// sequences of 400 keys and two tokens of each: not kept.)
// V's operand wants 8 keys of one component in a lane: a lane reads a word (8 components) of 8 keys and v_perm pairs their
// bytes.  Tiles come by LDS DMA into a ring of each wave's own, one or two ahead and waited for by their number, no barrier.
//
// Work is cut on the device, where the lengths are.  A unit is a tile of rows of one sequence and key head with the keys that
// it sees; the units of all sequences stand one behind the other on a line of keys (each with a lead for what its start
// costs), which the launch's workgroups, as many as are resident at once, divide evenly.  A workgroup of 4 waves goes
// through its stretch of the line unit by unit; waves without rows of their own share the unit's keys.  What a workgroup
// has of a unit that others work on too goes to its slots in `work`, and k_merge4 joins the parts.
//
// 32 heads over 8 of 128: 64 sequences of 200 to 8192 keys (311 MB) 76 to 87 us, one of 131072 (151 MB) 46 (3.3 TB/s), 2048
// rows of a prompt over 8192 keys (240 GFLOP) 507 (470 TFLOP/s).  The first two are the arithmetic of three waves a SIMD (70
// percent issue) and units' starts, the last that of two (77 percent, the matrix cores busy 24).  Starts are dearer with many
// sequences, which each workgroup's first wave goes through 64 at a time: the same bytes take 98 us in 256 of them, 121 in 512,
// 165 in 1024.  Scalar registers do not suffice: 146 to 173 are put away in lanes of vector registers, and about 20 brought
// back for each tile.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "dma_tile.h"
#include "kv4.h"
#include "lanes.h"
#include "quant4.h"

namespace {

using st::Cache;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// The three that follow were timed over 20 shapes, of 1 to 512 sequences and 1 to 2048 new tokens; us where it matters.
//
// Of the line for a workgroup at least: at 128, 256 and 512 one sequence of 128 keys takes 10.2, 10.5 and 10.5, 12 with 5 tokens
// each 24.4, 23.2 and 28.0, the others the same to 4 percent.
constexpr int MIN_STRETCH = 256;
// What a unit's start costs (finding it, its rows, its first loads, its end), in keys: at 256, 512 and 1024, 64 ragged sequences
// take 92.8, 87.0 and 88.9, 512 of them 138, 121 and 123, 12 with 5 tokens each 23.6, 23.2 and 26.9, 16 tokens of each of 64 213, 190
// and 201; only prompts alone would have it smaller (300 tokens over 3000 keys 69.4, 76.4 and 75.5).
constexpr int LEAD = 512;
// Units of up to so many keys are not shared among workgroups, as a merge would cost more: at 0, 512 and 2048, one sequence of 128
// keys takes 12.2, 10.5 and 10.4, 64 of 400 27.6, 21.2 and 21.3, 64 ragged ones 87.2, 87.0 and 87.9, 12 with 5 tokens each 23.4, 23.2 and
// 37.1, 6 prompts of 500 tokens 183, 184 and 222.
constexpr int WHOLE = 512;
constexpr int MAX_GROUPS = 1024;  // workgroups of a launch
constexpr int64_t MAX_ROWS = 1 << 26;  // rows times heads: no more units than that lie on the line, whose prefix sums then fit (load)
constexpr float BASE = 7.f, MOST_X = 32768.f;  // p aV is set to 2^7 at most, and may grow to 2^15
// Scales below 2^-86 count as that for the reference, so that p is 2^93 at most when it is set; it may grow until a tile's sum
// passes 2^101 (2^25 tiles stay within f32).
constexpr float MIN_E = -86.f, MOST_SUM = 0x1p101f;
// The part |b8| of a value counts for the reference too, 2^24 times less: p |b8| is set to 2^31 at most, and may grow until a tile's
// sum of p b8 passes 2^60.  Only vectors of components that are nearly equal (|b8| above 2^24 aV) are set by it.
constexpr float OFFSET = 0x1p-24f, MOST_LOW = 0x1p60f;

// What k_merge4 joins: a unit's rows, the first of them head `head` of token `token`; the first part is in the odd slot of the
// workgroup that this stands under, the others in the even slots of those behind it.
struct Joint {
    int parts, rows, token, head;
};

// Once the values of a tile pass 2^40 in the reference, a wave counts the unit's values in 2^40: p aV at 2^7 would put p itself near
// the end of f32's range (scales of 2^120: 2^-113, so that weights 2^12 below the largest were dropped).
constexpr float LARGE = 40.f, MOST_VALUE = 0x1p40f;
constexpr float ROOM = 10.f;  // a power of two that a unit's parts are no more than (MAX_GROUPS)

struct AttnArgs {
    Cache c;
    const void *q;
    void *out;
    float *lse;
    const int32_t *q_start, *kv_len;
    float *part_o;    // [2 groups, part_rows, hd] sums of parts of units
    float2 *part_ml;  // [2 groups, part_rows] their references and totals
    Joint *joints;    // [groups]
    int64_t q_stride;
    float scale2;  // scale log2 e
    int32_t n, hq, dtype, causal, window, one, groups, part_rows;
    int32_t share, cap;      // query heads of a key head, tokens of a table's row
    int32_t per, tile_rows;  // tokens (0: less than one) and rows of a tile
    int32_t lead;            // of each unit on the line
    int32_t most, small;     // the most keys that a tile sees; whether the line's positions fit 32 bits
    float inv_share, inv_groups;
    bool vec_q, vec_out;
};

// A value that is the same in every lane, in a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// x / y for quotients below 2^22: the f32 quotient is off by one at most.
__device__ __forceinline__ int quotient(int64_t x, int64_t y) {
    int q = (int)((float)x * __builtin_amdgcn_rcpf((float)y));
    const int64_t r = x - (int64_t)q * y;
    q += r >= y ? 1 : r < 0 ? -1 : 0;
    return q;
}

// What the line's position needs of 64 sequences.
struct Rows {
    int64_t upto[64], head[64];  // the line up to a sequence's end from the first of the 64 on, and of one of its heads
    int first[64], rows[64], len[64], tiles[64];
};

// What a workgroup does next: keys cut0 .. cut1 of a unit (none: it is done).  `parts`: of how many workgroups the unit is, where
// this one has its first part and not all of it, else 0.
struct Task {
    int cut0, cut1, keys, first, rows, len, head, tile, me, parts, s;
};
constexpr int TASK_WORDS = sizeof(Task) / 4;

// The line of keys, how units lie on it, and the workgroup's stretch of it.  Its first wave's.
struct Line {
    const AttnArgs &a;
    Rows &m;
    int lane;
    // `m` holds the 64 sequences from s0 on, `before` the line before them, `inside` theirs.
    int64_t s0 = 0, before = 0, inside = 0, length = 0, stretch = 0;
    int64_t at = 0, from = 0, to = 0, me = 0;
    int slot = 0;  // of the launch's workgroups, those without a stretch too

    __device__ __forceinline__ Line(const AttnArgs &args, Rows &mem, int lane_) : a(args), m(mem), lane(lane_) {}

    __device__ __forceinline__ void lay() {
        for (;; s0 += 64) {
            load();
            length += inside;
            if (s0 + 64 >= a.c.nseq) break;
        }
        // length / groups, not less: the f32 product is within 2^-22 of it.
        int64_t each = (int64_t)((float)length * a.inv_groups);
        each += (each >> 20) + 1;
        stretch = max((each + 127) & ~(int64_t)127, (int64_t)MIN_STRETCH);
        if (s0 > 0) s0 = 0, load();
    }

    // The line's part of a sequence's first j tiles of `tiles`: their leads and their keys (an upper bound where a window or rows
    // without keys make it less; a tile has one at least, so that each is some workgroup's).
    __device__ __forceinline__ int64_t part_of(int j, int tiles, int rows, int len) const {
        const int base = max(len - rows, 0), all = base + rows, most = a.most;
        const int64_t leads = (int64_t)j * a.lead;
        if (!a.causal || a.per == 0 || tiles == 1) return leads + (int64_t)j * min(all, most);
        // Tile i ends at token min((i + 1) per, rows) and sees base + that many keys, `most` of them.
        int64_t sum = leads;
        if (j == tiles) sum += min(all, most), j--;
        const int64_t grow = min(j, most > base ? (most - base) / a.per : 0);
        return sum + grow * base + a.per * (grow * (grow + 1) / 2) + (j - grow) * most;
    }

    __device__ __forceinline__ void load() {
        int first = 0, rows = 0, len = 0, tiles = 0;
        int64_t head = 0;
        if (s0 + lane < a.c.nseq) {
            const int64_t s = s0 + lane;
            const int next = a.q_start[s + 1];
            first = min(max(a.q_start[s], 0), a.n);
            len = max(a.kv_len[s], 0);
            rows = max(min(max(next, 0), a.n) - first, 0);
        }
        int64_t upto;
        if (a.small && !__any(rows > a.per)) {  // a tile each at most, and 32 bits suffice: a decoding step
            tiles = rows > 0 ? 1 : 0;
            head = tiles ? min(max(len, rows), a.most) + a.lead : 0;
            upto = st::wave_incl_scan((int)head * a.c.hkv);
        } else {
            tiles = a.per ? (rows + a.per - 1) / a.per : (int)(((int64_t)rows * a.share + a.tile_rows - 1) / a.tile_rows);
            if (tiles > 0) head = part_of(tiles, tiles, rows, len);
            // Prefix sums in two parts: 64 times 25 bits, and the rest of what is 2^26 units of 2^30 keys and a lead at most.
            const int64_t here = head * a.c.hkv;
            const int lo = st::wave_incl_scan((int)(here & 0x1FFFFFF)), hi = st::wave_incl_scan((int)(here >> 25));
            upto = ((int64_t)(uint32_t)hi << 25) + lo;
        }
        inside = st::lane_value64(upto, 63);
        m.upto[lane] = upto, m.head[lane] = head;
        m.first[lane] = first, m.rows[lane] = rows, m.len[lane] = len, m.tiles[lane] = tiles;
    }

    // A unit on the line.
    struct Unit {
        int64_t s, start;  // sequence, position of its first key
        int keys, first, rows, len, tiles, head, tile;
    };

    // Fills in `u` what goes by its sequence (the l-th of the 64): returns its first position, and the line's part of a head.
    __device__ __forceinline__ int64_t take(int l, Unit &u, int64_t &head) const {
        u.s = s0 + l;
        u.first = uniform(m.first[l]), u.rows = uniform(m.rows[l]), u.len = uniform(m.len[l]), u.tiles = uniform(m.tiles[l]);
        head = st::lane_value64(m.head[l], 0);
        return before + st::lane_value64(m.upto[l], 0) - head * a.c.hkv;
    }

    __device__ __forceinline__ void place(Unit &u, int64_t head_start, int tile) const {
        u.tile = uniform(tile);
        if (u.tiles == 1) {
            u.start = head_start + a.lead, u.keys = min(max(u.len, u.rows), a.most);
            return;
        }
        const int64_t ahead = part_of(u.tile, u.tiles, u.rows, u.len);
        u.start = head_start + ahead + a.lead;
        u.keys = uniform((int)(part_of(u.tile + 1, u.tiles, u.rows, u.len) - ahead) - a.lead);
    }

    // The unit that position `x` belongs to (not before the last one asked for).
    __device__ __forceinline__ Unit unit_at(int64_t x) {
        while (x >= before + inside) before += inside, s0 += 64, load();
        const int l = __ffsll((unsigned long long)__ballot(before + m.upto[lane] > x)) - 1;
        Unit u;
        int64_t each;
        const int64_t base = take(l, u, each);
        u.head = uniform(quotient(x - base, each));
        const int64_t off = x - base - u.head * each;
        int lo = 0, hi = u.tiles - 1;  // the last tile whose lead does not begin behind `off`
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (part_of(mid, u.tiles, u.rows, u.len) <= off)
                lo = mid;
            else
                hi = mid - 1;
        }
        place(u, base + u.head * each, lo);
        return u;
    }

    // Where a stretch that ends at position `end` ends within a unit: at a multiple of 128 of its keys.
    __device__ __forceinline__ int cut(const Unit &u, int64_t end) const {
        const int64_t x = end - u.start;
        if (x <= 0) return 0;
        return u.keys <= WHOLE ? u.keys : (int)min((x + 127) & ~(int64_t)127, (int64_t)u.keys);
    }

    // The workgroup's stretch.  Neighbouring ones go to one XCD (workgroups go round the 8 of them): units of a head share pages.
    __device__ __forceinline__ void begin() {
        lay();
        const int used = uniform(quotient(length + stretch - 1, stretch)), each = (used + 7) / 8, row = blockIdx.x >> 3;
        me = (int64_t)(blockIdx.x & 7) * each + row;
        if (row >= each || me >= used) {
            slot = row < each ? (int)me : (int)blockIdx.x;
            return;
        }
        slot = (int)me;
        from = at = me * stretch;
        to = min(from + stretch, length);
    }

    __device__ __forceinline__ void next(Task &t) {
        Unit u = {};
        int cut0 = 0, cut1 = 0, parts = 0;
        while (at < to && cut0 == cut1) {
            u = unit_at(at);
            at = u.start + u.keys;
            cut0 = uniform(cut(u, from)), cut1 = uniform(cut(u, to));
        }
        if (cut0 == 0 && cut1 > 0 && cut1 < u.keys) {
            const int last = quotient(u.start + u.keys - 1, stretch);
            // The last one's share may be empty: its keys went to the one before.
            parts = uniform(last - (int)me + (cut(u, last * stretch) < u.keys ? 1 : 0));
        }
        if (lane == 0) t = {cut0, cut1, u.keys, u.first, u.rows, u.len, u.head, u.tile, (int)me, parts, (int)u.s};
    }
};

// The rows of a task's tile (a token's heads side by side, from head rem0 of token tok0 on) and the first key that they see.
struct Span {
    int rows, tok0, rem0, base, lo;
    float inv_share;

    __device__ __forceinline__ Span(const AttnArgs &a, const Task &u) : inv_share(a.inv_share) {
        const int row0 = u.tile * a.tile_rows;
        rows = min(a.tile_rows, u.rows * a.share - row0);
        tok0 = a.per ? u.tile * a.per : uniform(quotient(row0, a.share)), rem0 = a.per ? 0 : row0 - tok0 * a.share;
        base = u.len - u.rows + tok0;  // position of the first row (negative: more rows than tokens)
        lo = a.window > 0 ? (int)(max((int64_t)0, (int64_t)base + 1 - a.window) & ~63) : 0;  // down to a tile's start
    }
    __device__ __forceinline__ int token_of(int x) const { return (int)(((float)(rem0 + x) + 0.5f) * inv_share); }  // of row x, from tok0 on
    __device__ __forceinline__ int pos_of(const AttnArgs &a, const Task &u, int x) const { return a.causal ? base + token_of(x) : u.len - 1; }
    // Element offset of row x in q, and its index in out's [n, hq].
    __device__ __forceinline__ int64_t q_at(const AttnArgs &a, const Task &u, int x, int hd) const {
        const int token = token_of(x);
        return (int64_t)(u.first + tok0 + token) * a.q_stride + (int64_t)(u.head * a.share + rem0 + x - token * a.share) * hd;
    }
    __device__ __forceinline__ int64_t row_at(const AttnArgs &a, const Task &u, int x) const {
        const int token = token_of(x);
        return (int64_t)(u.first + tok0 + token) * a.hq + u.head * a.share + rem0 + x - token * a.share;
    }
};

// The task from LDS, each word to a scalar register.
__device__ __forceinline__ Task read_task(const Task &t, int lane) {
    const int word = ((const int *)&t)[min(lane, TASK_WORDS - 1)];
    Task u;
#pragma unroll
    for (int i = 0; i < TASK_WORDS; i++) ((int *)&u)[i] = st::lane_value(word, i);
    return u;
}

__device__ __forceinline__ void load_q(const AttnArgs &a, int64_t at, float (&x)[8]) {
    if (a.dtype == ST_F32)
        st::load8((const float *)a.q + at, a.vec_q, x);
    else if (a.dtype == ST_F16)
        st::load8((const _Float16 *)a.q + at, a.vec_q, x);
    else
        st::load8((const __bf16 *)a.q + at, a.vec_q, x);
}

// x 2^d, d a whole number (or infinite).
__device__ __forceinline__ float times_2_to(float x, float d) { return __builtin_amdgcn_ldexpf(x, (int)fminf(fmaxf(d, -1000.f), 1000.f)); }

// The largest component's exponent in `most` (0 where it is 0 or not finite): a row is scaled by 2^(15 - it).
__device__ __forceinline__ int lift_of(float most) {
    return most > 0.f && __builtin_isfinite(most) ? 15 - __builtin_amdgcn_frexp_expf(most) : 0;
}

// A row's sums to its output and log-sum-exp: v and l in units of 2^top, l at most 1.
struct Ending {
    float inv, shift, lse;
    __device__ __forceinline__ Ending(const AttnArgs &a, float top, float l) {
        const float units = a.one ? fmaxf(top, 0.f) : top;  // (the phantom weighs 1)
        shift = a.one ? top - units : 0.f;
        const float sum = times_2_to(l, shift) + (a.one ? __builtin_amdgcn_exp2f(-units) : 0.f);
        inv = sum == 0.f ? 0.f : 1.f / sum;
        lse = sum == 0.f ? -INFINITY : (units + __builtin_amdgcn_logf(sum)) * 0.693147180559945309f;
    }
    __device__ __forceinline__ float operator()(float v) const { return times_2_to(v * inv, shift); }
};

// The waves' sums of a tile's rows, each against the wave's own reference, joined: to out, or to the workgroup's slot of a
// unit that others work on too.  `sums` [4 waves][wave_rows][hd + 4], `ml` [4][wave_rows]; `sharing` waves have the same rows.
//
// References follow the values' sizes and say little about weights: a wave whose values are all 0 is 2^86 and more below one
// with ordinary ones.  So the joined row is in units of its largest weight, times 4, which takes the weights' sum to 1 at most
// and the values' to no more than the largest value; references are whole, and so the factors powers of two.
template <int HD>
__device__ __forceinline__ void finish(const AttnArgs &a, const Task &u, const Span &span, const float *sums, const float2 *ml, int wave_rows,
                                       int sharing) {
    for (int i = threadIdx.x; i < span.rows * (HD / 8); i += 256) {
        const int y = i / (HD / 8), e = 8 * (i % (HD / 8)), w0 = y / wave_rows * sharing, z = y % wave_rows;
        float2 t[4];
        float top = -INFINITY, l = 0.f, v[8] = {};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            t[k] = ml[min(w0 + k, 3) * wave_rows + z];
            if (k >= sharing) t[k] = make_float2(-INFINITY, 0.f);
            top = fmaxf(top, t[k].x + __builtin_amdgcn_logf(t[k].y));
        }
        top = ceilf(top) + 2.f;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float d = t[k].x - top;  // (NaN where there is nothing)
            l += times_2_to(t[k].y, d);
            if (k < sharing) {
                float w[8];
                st::load8(sums + ((w0 + k) * wave_rows + z) * (HD + 4) + e, true, w);
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] += times_2_to(w[j], d);
            }
        }
        if (u.cut0 > 0 || u.cut1 < u.keys) {
            const int64_t slot = (2 * (int64_t)u.me + (u.cut0 == 0 ? 1 : 0)) * a.part_rows + y;
            st::store8(a.part_o + slot * HD + e, true, v);
            if (e == 0) a.part_ml[slot] = make_float2(top, l);
            continue;
        }
        const int64_t row = span.row_at(a, u, y);
        const Ending ending(a, top, l);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = ending(v[j]);
        if (a.dtype == ST_F32)
            st::store8((float *)a.out + row * HD + e, a.vec_out, v);
        else if (a.dtype == ST_F16)
            st::store8((_Float16 *)a.out + row * HD + e, a.vec_out, v);
        else
            st::store8((__bf16 *)a.out + row * HD + e, a.vec_out, v);
        if (a.lse && e == 0) a.lse[row] = ending.lse;
    }
}

// The head's components in blocks of 128, 64 or 32: lane column c of a block of width W reads W / 16 components from
// W / 16 c on, which lie in one word.
constexpr int block_width(int hd, int b) {
    return b == 0 ? (hd >= 128 ? 128 : hd >= 64 ? 64 : 32) : hd == 96 ? 32 : hd == 192 ? 64 : hd == 256 ? 128 : 0;
}
constexpr int blocks_of(int hd) { return block_width(hd, 1) ? 2 : 1; }

// 16 bytes a lane from scalar base + lane offset, or from a lane's address, to LDS from `to` on.  In assembly, so that the
// compiler does not wait for every load in flight before any LDS read: a tile's loads are waited for by their number.
__device__ __forceinline__ void bring(const void *base, uint32_t off, uint32_t to) {
    uint32_t saved;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %3\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %1, %2\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "v"(off), "s"(base), "s"(to)
        : "memory");
}
__device__ __forceinline__ void bring(const void *at, uint32_t to) {
    uint32_t saved;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %2\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %1, off\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "v"(at), "s"(to)
        : "memory");
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

// O^T += V^T P^T for 32 keys: `word(b, i)` is this lane's word of block b of the i-th of its 8 keys, ph (and pr, the weights'
// second parts) its 8 weights of each 16 rows.
template <int HD, int WEIGHTS, int RT, class Word>
__device__ __forceinline__ void weigh_values(const Taker &take, const Word &word, const h8 (&ph)[RT], const h8 (&pr)[WEIGHTS == 2 ? RT : 1], int col,
                                             f4 (&o)[RT][HD / 16]) {
#pragma unroll
    for (int b = 0; b < blocks_of(HD); b++) {
        constexpr int first = block_width(HD, 0) / 16;
        const int width = block_width(HD, b);
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = word(b, i);
#pragma unroll
        for (int i = 0; i < width / 32; i++) {
            const int byte = width == 128 ? i : width == 64 ? 2 * (col & 1) + i : col & 3;
            const uint32_t sel = 0x0c000c00u | (uint32_t)(4 + byte) << 16 | (uint32_t)byte;
            const uint32_t x0 = __builtin_amdgcn_perm(w[1], w[0], sel), x1 = __builtin_amdgcn_perm(w[3], w[2], sel);
            const uint32_t x2 = __builtin_amdgcn_perm(w[5], w[4], sel), x3 = __builtin_amdgcn_perm(w[7], w[6], sel);
            const h8 even = as_h8(take.lower(x0), take.lower(x1), take.lower(x2), take.lower(x3));
            const h8 odd = as_h8(take.upper(x0), take.upper(x1), take.upper(x2), take.upper(x3));
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                f4 &e = o[rt][b * first + 2 * i], &d = o[rt][b * first + 2 * i + 1];
                e = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, ph[rt], e, 0, 0, 0);
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, ph[rt], d, 0, 0, 0);
                if constexpr (WEIGHTS == 2) {
                    e = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, pr[rt], e, 0, 0, 0);
                    d = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, pr[rt], d, 0, 0, 0);
                }
            }
        }
    }
}

// This lane's byte offset in a row of codes of its word of block b.
template <int HD>
__device__ __forceinline__ int word_at(int b, int col) {
    const int width = block_width(HD, b), start = b ? block_width(HD, 0) : 0;
    return start / 2 + 4 * (width == 128 ? col : width == 64 ? col >> 1 : col >> 2);
}

// Puts o [col = row][components] and `low`, which goes to every component of the row, to a row of a wave's sums.
template <int HD>
__device__ __forceinline__ void put_sums(float *row, const f4 (&o)[HD / 16], float low, int g) {
#pragma unroll
    for (int b = 0; b < blocks_of(HD); b++) {
        constexpr int first = block_width(HD, 0) / 16;
        const int per = block_width(HD, b) / 16, start = b ? block_width(HD, 0) : 0;
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int j = 0; j < per; j++) row[start + per * (4 * g + r) + j] = o[b * first + j][r] + low;
    }
}

// A wave's ring of tiles in LDS.  A tile (32 keys: their codes and (scale, lo) pairs, in two halves of 16 keys, which a page may
// end between) is brought by DMA in chunks of 16 bytes: of K, then of V, then the pairs of K and of V.  A chunk's place is
// 16 bytes times its number; which chunk of memory it is, is the lane's choice:
//  - K of 128 and 256 components: in the order that lanes read their fragments in (lane (col, g) key col's 16 bytes from
//    piece g, or 2 g + i, on), which no bank is hit twice by; else key by key;
//  - V: rows in the order 0 4 8 12 1 5 .., so that the four keys that a read takes lie side by side.
template <int HD>
struct Ring {
    static constexpr int NW = HD / 32;
    static constexpr int PER_KEY = HD / 32, HALF = 16 * PER_KEY;                    // chunks
    static constexpr int LOADS = (2 * HD + 32 + 63) / 64, BYTES = 1024 * LOADS;    // of a tile
    static constexpr bool EVEN = HD == 128 || HD == 256;                            // a load is of one half of K or of V
    static constexpr int PAIRS = 32 * HD;                                           // byte offset of the pairs

    // Source byte offset of chunk `n` of a half of K or V.
    static __device__ __forceinline__ int source(int n, bool v) {
        if (v) {
            const int slot = n / PER_KEY;
            return (4 * (slot & 3) + (slot >> 2)) * (HD / 2) + 16 * (n % PER_KEY);
        }
        if (HD == 128) return (n & 15) * (HD / 2) + 16 * (n >> 4);
        if (HD == 256) return (n & 15) * (HD / 2) + 16 * (2 * ((n >> 4) & 3) + (n >> 6));
        return n / PER_KEY * (HD / 2) + 16 * (n % PER_KEY);
    }

    // This lane's words of K's half `half`.
    static __device__ __forceinline__ void k_words(const char *tile, int half, int lane, uint32_t (&w)[NW]) {
        typedef uint32_t v2 __attribute__((ext_vector_type(2)));
        const int col = lane & 15, g = lane >> 4;
        if constexpr (EVEN) {
#pragma unroll
            for (int i = 0; i < NW; i += 4) {
                const u4 x = *(const u4 *)(tile + 16 * (HALF * half + 16 * i + lane));
                w[i] = x[0], w[i + 1] = x[1], w[i + 2] = x[2], w[i + 3] = x[3];
            }
        } else {
            const char *p = tile + 16 * HALF * half + col * (HD / 2) + g * (HD / 8);
            if constexpr (NW % 2 == 0) {
#pragma unroll
                for (int i = 0; i < NW; i += 2) {
                    const v2 x = *(const v2 *)(p + 4 * i);
                    w[i] = x[0], w[i + 1] = x[1];
                }
            } else {
#pragma unroll
                for (int i = 0; i < NW; i++) w[i] = *(const uint32_t *)(p + 4 * i);
            }
        }
    }

    // The (scale, lo) pairs of keys (or values) 4 g + 2 i and the next of half `half`.
    static __device__ __forceinline__ float4 pairs(const char *tile, bool v, int half, int i, int g) {
        return *(const float4 *)(tile + PAIRS + 256 * v + 128 * half + 32 * g + 16 * i);
    }
};

// A wave-uniform value in scalar registers of its own.  Kernel arguments arrive eight or sixteen words at a time, and where
// scalar registers are short the compiler puts away and brings back all of those for one that a loop needs.
template <class T>
__device__ __forceinline__ T alone(T x) {
    asm("" : "+s"(x));
    return x;
}

template <int HD, int PARTS, int WEIGHTS, int RT>
__global__ __launch_bounds__(256, (RT == 1 && HD <= 128 ? 3 : 2)) void k_attention4(const AttnArgs a) {
    using R = Ring<HD>;
    constexpr int NW = HD / 32, WAVE_ROWS = 16 * RT, LDO = HD + 4, STAGES = RT == 1 ? 2 : 3;
    constexpr int RING = 4 * STAGES * R::BYTES, SUMS = 4 * WAVE_ROWS * LDO * 4;
    __shared__ __align__(16) char mem[RING > SUMS ? RING : SUMS];  // the waves' rings, then their sums
    __shared__ float2 ml[4][WAVE_ROWS];
    __shared__ Rows row_mem;
    __shared__ Task task;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const Cache &c = a.c;
    const Taker take;
    char *ring = mem + wave * STAGES * R::BYTES;
    const uint32_t ring_at = uniform((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char *)ring);
    Line line(a, row_mem, lane);
    Joint joint = {};
    if (wave == 0) line.begin();

    for (;;) {
        if (wave == 0) line.next(task);
        __syncthreads();
        const Task u = read_task(task, lane);
        if (u.cut0 == u.cut1) {
            if (threadIdx.x == 0 && a.part_rows) a.joints[line.slot] = joint;
            return;
        }
        const Span span(a, u);
        if (u.parts > 1) joint = {u.parts, span.rows, u.first + span.tok0, u.head * a.share + span.rem0};
        const int rows = uniform(span.rows), cap = a.cap;
        const int groups = (rows + WAVE_ROWS - 1) / WAVE_ROWS, sharing = groups == 1 ? 4 : groups == 2 ? 2 : 1;
        const int group = wave / sharing, turn = wave % sharing;
        const bool busy = group < groups;

        // This lane's row of each 16, and the positions of the group's first and last.
        int pos[RT];
        const int first_row = group * WAVE_ROWS, last_row = min(first_row + WAVE_ROWS, rows) - 1;
        const int pos_first = uniform(span.pos_of(a, u, first_row)), pos_last = uniform(span.pos_of(a, u, last_row));

        // The group's keys of this part: those that its first row may see up to those of its last, within the table.
        int begin = span.lo + u.cut0, end = min(pos_last + 1, cap);
        if (u.cut1 < u.keys) end = min(end, span.lo + u.cut1);
        if (a.window > 0) begin = max(begin, (int)(max((int64_t)0, (int64_t)pos_first + 1 - a.window) & ~31));
        begin = uniform(begin), end = uniform(end);
        const int first_key = uniform(begin + 32 * turn), step = 32 * sharing;
        const int count = uniform(busy && c.pages > 0 && end > first_key ? (end - first_key + step - 1) / step : 0);

        // Pages of the next 32 tiles' halves, a half a lane: -1 one outside the cache, 0 (not looked at) behind the end.
        const int page_rows = alone(c.hkv * c.page), head_row = alone(u.head * c.page), page_mask = alone(c.page - 1), window = alone(a.window);
        const uint8_t *const k_codes = alone(c.k_codes), *const v_codes = alone(c.v_codes);
        const float2 *const k_scales = alone(c.k_scales), *const v_scales = alone(c.v_scales);
        int entries = 0, entries_to = 0;
        uint32_t bad = 0;  // of the tiles in the ring, two bits each
        auto bring_tile = [&](int it, int slot) {
            if (it >= entries_to) {
                const int key = first_key + (it + (lane >> 1)) * step + 16 * (lane & 1);
                entries = 0;
                if (key < end) {
                    const int p = c.table[(int64_t)u.s * c.max_pages + (key >> c.page_log2)];
                    entries = p >= 0 && p < c.pages ? p : -1;
                }
                entries_to = it + 32;
            }
            const int key = first_key + it * step, i = 2 * (it + 32 - entries_to);
            const int p0 = st::lane_value(entries, i), p1 = st::lane_value(entries, i + 1);
            bad = (bad & ~(3u << (2 * slot))) | ((p0 < 0 ? 1u : 0u) | (p1 < 0 ? 2u : 0u)) << (2 * slot);
            const int64_t row_0 = (int64_t)max(p0, 0) * page_rows + (head_row + (key & page_mask));
            const int64_t row_1 = (int64_t)max(p1, 0) * page_rows + (head_row + ((key + 16) & page_mask));
            const uint32_t to = ring_at + slot * R::BYTES;
            const int64_t b0 = row_0 * (HD / 2), b1 = row_1 * (HD / 2);
#pragma unroll
            for (int i = 0; i < R::LOADS; i++) {
                if (R::EVEN && i < HD / 32) {  // one half of K or V
                    const bool v = i >= HD / 64;
                    const int j = v ? i - HD / 64 : i, half = 64 * j / R::HALF;
                    bring((v ? v_codes : k_codes) + (half ? b1 : b0), R::source(64 * j % R::HALF + lane, v), to + 1024 * i);
                } else {
                    int n = 64 * i + lane;
                    const char *from;
                    if (n < 2 * HD) {
                        const bool v = n >= HD;
                        n -= v ? HD : 0;
                        from = (const char *)(v ? v_codes : k_codes) + (n >= R::HALF ? b1 : b0) + R::source(n % R::HALF, v);
                    } else {
                        n = (n - 2 * HD) & 31;  // lanes without a chunk of their own repeat one into the tile's padding
                        from = (const char *)(n >= 16 ? v_scales : k_scales) + (n & 8 ? row_1 : row_0) * 8 + 16 * (n & 7);
                    }
                    bring(from, to + 1024 * i);
                }
            }
        };
#pragma unroll
        for (int i = 0; i < STAGES; i++)
            if (i < count) bring_tile(i, i);

        h8 qh[RT][NW], ql[PARTS == 2 ? RT : 1][PARTS == 2 ? NW : 1];
        float unscale[RT], qsum[RT], qsum8[RT];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const int r = first_row + 16 * rt + col;
            pos[rt] = span.pos_of(a, u, min(r, rows - 1));
            float x[NW][8];
            float most = 0.f, sum = 0.f;
            bool finite = true;
#pragma unroll
            for (int w = 0; w < NW; w++)
#pragma unroll
                for (int i = 0; i < 8; i++) x[w][i] = 0.f;
            if (busy && r < rows) {
                const int64_t from = span.q_at(a, u, r, HD) + g * (HD / 4);
#pragma unroll
                for (int w = 0; w < NW; w++) load_q(a, from + 8 * w, x[w]);
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
            const int e = lift_of(most);
            unscale[rt] = __builtin_amdgcn_ldexpf(a.scale2, -e);
            qsum[rt] = a.scale2 * sum, qsum8[rt] = 8.f * qsum[rt];
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

        f4 o[RT][HD / 16];
        float ref[RT], total[RT], low[RT];  // sums in units of 2^ref
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            ref[rt] = -INFINITY, total[rt] = low[rt] = 0.f;
#pragma unroll
            for (int j = 0; j < HD / 16; j++) o[rt][j] = f4{0.f, 0.f, 0.f, 0.f};
        }
        bool large = false;  // values count in 2^LARGE
        auto process = [&](char *tile, int it, int bad_halves) {
            const int kt = first_key + it * step, key0 = kt + 4 * g;
            const bool masked = kt + 31 > pos_first || kt + 31 >= end || (window > 0 && kt <= pos_last - window);
            bool careful = false;
            if (masked || bad_halves || large) {
                // What lies behind the end counts nothing, whatever it holds; keys on a page outside the cache are NaN to the
                // rows that see them; and a value that is not finite must not reach the rows that do not see it, as 0 times it.
                const int k = lane & 31;
                const bool gone = bad_halves & (k & 16 ? 2 : 1);
                float2 *kp = (float2 *)(tile + R::PAIRS) + k, *vp = kp + 32;
                const float2 v = *vp;
                if (gone) *kp = make_float2(NAN, NAN);
                if (gone || kt + k >= end)
                    *vp = make_float2(0.f, 0.f);
                else if (large)
                    *vp = make_float2(times_2_to(v.x, -LARGE), times_2_to(v.y, -LARGE));
                careful = __any(!gone && kt + k < end && !__builtin_isfinite(v.x + v.y));
            }
            // Scores of the tile less `shift`, in log2.
            auto scores = [&](const char *tile, const float (&shift)[RT], float (&z)[RT][2][4]) {
                f4 s[RT][2];
#pragma unroll
                for (int rt = 0; rt < RT; rt++) s[rt][0] = s[rt][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    uint32_t kw[NW];
                    R::k_words(tile, i, lane, kw);
#pragma unroll
                    for (int w = 0; w < NW; w++) {
                        const h8 k8 = take.codes8(kw[w]);
#pragma unroll
                        for (int rt = 0; rt < RT; rt++) {
                            s[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, qh[rt][w], s[rt][i], 0, 0, 0);
                            if constexpr (PARTS == 2) s[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, ql[rt][w], s[rt][i], 0, 0, 0);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int r = 0; r < 4; r += 2) {
                        const float4 y = R::pairs(tile, false, i, r / 2, g);
#pragma unroll
                        for (int rt = 0; rt < RT; rt++) {
                            z[rt][i][r] = __builtin_fmaf(y.x, __builtin_fmaf(s[rt][i][r], unscale[rt], qsum8[rt]), __builtin_fmaf(y.y, qsum[rt], -shift[rt]));
                            z[rt][i][r + 1] = __builtin_fmaf(y.z, __builtin_fmaf(s[rt][i][r + 1], unscale[rt], qsum8[rt]), __builtin_fmaf(y.w, qsum[rt], -shift[rt]));
                        }
                    }
                if (masked) {
#pragma unroll
                    for (int rt = 0; rt < RT; rt++) {
                        const int after = window > 0 ? pos[rt] - window : -1;
#pragma unroll
                        for (int i = 0; i < 2; i++)
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                const int key = key0 + 16 * i + r;
                                z[rt][i][r] = key <= pos[rt] && key > after ? z[rt][i][r] : -INFINITY;
                            }
                    }
                }
            };
            // p = 2^(z - R), p aV and the sum of p b8 of every row.  For the first tile, and where p aV would pass f16's range or p
            // or p b8 an f32's, the scores are taken again to set R: seldom, and the common tile holds no registers for it. (The
            // tile's p are no larger than their sum.)
            float p[RT][2][4], sum[RT], low_sum[RT];
            h8 ph[RT], pr[WEIGHTS == 2 ? RT : 1];
            auto weights = [&](const char *tile) {  // p aV in f16, rounded once
#pragma unroll
                for (int rt = 0; rt < RT; rt++) low_sum[rt] = 0.f;
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float4 y = R::pairs(tile, true, i, r / 2, g);
                        const float v = r & 1 ? y.z : y.x, v8 = __builtin_fmaf(8.f, v, r & 1 ? y.w : y.y);  // v8: what a code of 8 stands for
#pragma unroll
                        for (int rt = 0; rt < RT; rt++) {
                            low_sum[rt] = __builtin_fmaf(p[rt][i][r], v8, low_sum[rt]);
                            ph[rt][4 * i + r] = (_Float16)__builtin_fmaf(p[rt][i][r], v, 0.f);
                            if constexpr (WEIGHTS == 2) pr[rt][4 * i + r] = (_Float16)__builtin_fmaf(p[rt][i][r], v, -(float)ph[rt][4 * i + r]);
                        }
                    }
            };
            bool past = true;
            if (it > 0) {
                scores(tile, ref, p);
                float most_p = 0.f;
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    sum[rt] = 0.f;
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            p[rt][i][r] = __builtin_amdgcn_exp2f(p[rt][i][r]);
                            sum[rt] += p[rt][i][r];
                        }
                    most_p = fmaxf(most_p, sum[rt]);
                }
                weights(tile);
                h2 most_x = {};
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
#pragma unroll
                    for (int i = 0; i < 4; i++) most_x = __builtin_elementwise_max(most_x, h2{ph[rt][2 * i], ph[rt][2 * i + 1]});
                past = most_p > MOST_SUM || (float)most_x[0] > MOST_X || (float)most_x[1] > MOST_X;
                if (careful) {  // rows that see what is not finite are left alone: the others' references are as without it
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const float4 y = R::pairs(tile, true, i, r / 2, g);
                            const float v8 = __builtin_fmaf(8.f, r & 1 ? y.z : y.x, r & 1 ? y.w : y.y);
#pragma unroll
                            for (int rt = 0; rt < RT; rt++) past = past || (__builtin_isfinite(v8) && fabsf(p[rt][i][r] * v8) > MOST_LOW);
                        }
                } else {  // (infinities that cancel leave NaN; a sum of p that is NaN is the scores')
#pragma unroll
                    for (int rt = 0; rt < RT; rt++) past = past || (!(fabsf(low_sum[rt]) <= MOST_LOW) && sum[rt] == sum[rt]);
                }
            }
            if (__any(past)) {
                uint32_t from = uniform((uint32_t)(tile - mem));
                asm volatile("" : "+s"(from));  // read again, not kept
                char *again = mem + from;
                // The size of a value as the reference takes it, of its scale and its value for a code of 8.
                auto size_of = [](float v, float v8) { return fmaxf(v, fabsf(v8) * OFFSET); };
                float2 *const vp = (float2 *)(again + R::PAIRS) + 32 + (lane & 31);
                const float2 v = *vp;
                if (!large && __any(size_of(v.x, __builtin_fmaf(8.f, v.x, v.y)) >= MOST_VALUE)) {
                    large = true;
                    *vp = make_float2(times_2_to(v.x, -LARGE), times_2_to(v.y, -LARGE));
                    // What is summed up: p is larger by what values are less, as far as its own range allows.
#pragma unroll
                    for (int rt = 0; rt < RT; rt++) {
                        float all = fmaxf(total[rt], st::xor_lane(total[rt], 16, lane));
                        all = fmaxf(all, st::xor_lane(all, 32, lane));
                        const float up = fminf(fmaxf(100.f - (float)__builtin_amdgcn_frexp_expf(all), 0.f), LARGE);
                        ref[rt] -= up, total[rt] = times_2_to(total[rt], up), low[rt] = times_2_to(low[rt], up - LARGE);
#pragma unroll
                        for (int j = 0; j < HD / 16; j++)
#pragma unroll
                            for (int i = 0; i < 4; i++) o[rt][j][i] = times_2_to(o[rt][j][i], up - LARGE);
                    }
                }
                float zero[RT] = {};
                scores(again, zero, p);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    float m = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const float4 y = R::pairs(again, true, i, r / 2, g);
                            const float scale = r & 1 ? y.z : y.x, size = size_of(scale, __builtin_fmaf(8.f, scale, r & 1 ? y.w : y.y));
                            m = fmaxf(m, p[rt][i][r] + fmaxf(size > 0.f ? (float)__builtin_amdgcn_frexp_expf(size) : MIN_E, MIN_E));
                        }
                    m = fmaxf(m, st::xor_lane(m, 16, lane));
                    m = fmaxf(m, st::xor_lane(m, 32, lane));
                    m = fmaxf(ref[rt], ceilf(m) - BASE);
                    const float keep = ref[rt] - m;  // (NaN where there is nothing yet)
                    total[rt] = times_2_to(total[rt], keep), low[rt] = times_2_to(low[rt], keep);
#pragma unroll
                    for (int j = 0; j < HD / 16; j++)
#pragma unroll
                        for (int i = 0; i < 4; i++) o[rt][j][i] = times_2_to(o[rt][j][i], keep);
                    ref[rt] = m;
                    sum[rt] = 0.f;
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            // (A row without a reference sees nothing here: minus infinity less itself is no number.)
                            p[rt][i][r] = m == -INFINITY && p[rt][i][r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(p[rt][i][r] - m);
                            sum[rt] += p[rt][i][r];
                        }
                }
                weights(again);
            }
#pragma unroll
            for (int rt = 0; rt < RT; rt++) total[rt] += sum[rt];
            if (careful) {  // (a weight of 0 leaves even what is not a number out)
#pragma unroll
                for (int rt = 0; rt < RT; rt++) low_sum[rt] = 0.f;
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float4 y = R::pairs(tile, true, i, r / 2, g);
                        const float v8 = __builtin_fmaf(8.f, r & 1 ? y.z : y.x, r & 1 ? y.w : y.y);
#pragma unroll
                        for (int rt = 0; rt < RT; rt++) {
                            const bool none = p[rt][i][r] == 0.f;
                            low_sum[rt] = none ? low_sum[rt] : __builtin_fmaf(p[rt][i][r], v8, low_sum[rt]);
                            ph[rt][4 * i + r] = none ? (_Float16)0.f : ph[rt][4 * i + r];
                            if constexpr (WEIGHTS == 2) pr[rt][4 * i + r] = none ? (_Float16)0.f : pr[rt][4 * i + r];
                        }
                    }
            }
#pragma unroll
            for (int rt = 0; rt < RT; rt++) low[rt] += low_sum[rt];
            weigh_values<HD, WEIGHTS, RT>(take, [&](int b, int i) {  // keys 4 g .. of each half, whose rows lie in the order 0 4 8 12 1 ..
                return *(const uint32_t *)(tile + 16 * (HD + R::HALF * (i >> 2)) + (4 * (i & 3) + g) * (HD / 2) + word_at<HD>(b, col));
            }, ph, pr, col, o);
        };

        for (int it = 0, slot = 0; it < count; it++) {
            // This tile's loads are over when only those of the STAGES - 1 behind it are under way (near the end: when none is).
            if (it + STAGES <= count)
                dma::wait_vm<(STAGES - 1) * R::LOADS>();
            else
                dma::wait_vm<0>();
            asm volatile("" ::: "memory");
            process(ring + slot * R::BYTES, it, (bad >> (2 * slot)) & 3);
            __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the tile's last reads are over before it is overwritten
            if (it + STAGES < count) bring_tile(it + STAGES, slot);
            slot = slot + 1 == STAGES ? 0 : slot + 1;
        }

        if (large) {
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                low[rt] = times_2_to(low[rt], LARGE);
#pragma unroll
                for (int j = 0; j < HD / 16; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[rt][j][i] = times_2_to(o[rt][j][i], LARGE);
            }
        }

        // The sums of the waves that share rows, each against the wave's own reference, meet in LDS.
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            total[rt] += st::xor_lane(total[rt], 16, lane);
            total[rt] += st::xor_lane(total[rt], 32, lane);
            low[rt] += st::xor_lane(low[rt], 16, lane);
            low[rt] += st::xor_lane(low[rt], 32, lane);
            // A row whose own token lies past the table, or that sees a token of a cache without pages (its own at least).
            if (pos[rt] >= (c.pages == 0 ? 0 : cap)) total[rt] = NAN;
            if (g == 0) ml[wave][16 * rt + col] = make_float2(ref[rt], total[rt]);
        }
        __syncthreads();  // every ring is read
        float *sums = (float *)mem;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) put_sums<HD>(sums + (wave * WAVE_ROWS + 16 * rt + col) * LDO, o[rt], low[rt], g);
        __syncthreads();
        finish<HD>(a, u, span, sums, &ml[0][0], WAVE_ROWS, sharing);
        __syncthreads();  // the sums are read before the rings are filled again
    }
}

// Joins the parts of units that several workgroups worked on: out = sum 2^(M_i - M) O_i / sum 2^(M_i - M) l_i over a row's parts,
// M 2^ROOM above the largest, so that the sums pass neither 1 nor the largest value.  (l_i is between 1/8 and 1, so what is below
// 2^-126 here weighs less than 2^-113.)
// Workgroup (i, j) has the unit that begins in the launch's workgroup i, and WAVES waves to each row of its j-th 4 / WAVES, and of
// those as many further on as the launch has in all.
template <int HD, int WAVES>
__global__ __launch_bounds__(256) void k_merge4(const AttnArgs a) {
    constexpr int LANES = HD / 4, GROUPS = 64 * WAVES / LANES, TEAMS = 4 / WAVES;
    __shared__ float weights[TEAMS][MAX_GROUPS + 8];
    __shared__ float red[TEAMS][GROUPS][HD], stat[8];
    const Joint joint = a.joints[blockIdx.x];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), team = wave / WAVES;
    const int me = threadIdx.x - team * 64 * WAVES, rows = min(joint.rows, a.part_rows), parts = min(joint.parts, MAX_GROUPS);
    if (parts < 2) return;
    float *weight = weights[team];
    for (int y = blockIdx.y * TEAMS + team; y < rows; y += gridDim.y * TEAMS) {  // (with four waves a row all of the workgroup's)
        auto slot = [&](int i) { return (2 * (int64_t)min((int)blockIdx.x + i, a.groups - 1) + (i == 0 ? 1 : 0)) * a.part_rows + y; };
        // The first parts' sums are under way while their weights are found (12 sequences with 5 tokens each 23.9 to 23.0 us, a
        // prompt 531 to 528).
        const int gr = me / LANES, e = 4 * (me % LANES);
        float4 x[8];
        auto load = [&](int i0) {
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (k == 0 || k * GROUPS < parts) x[k] = *(const float4 *)(a.part_o + slot(min(i0 + k * GROUPS, parts - 1)) * HD + e);
        };
        load(gr);
        float m = -INFINITY, l = 0.f;
        for (int i = me; i < parts; i += 64 * WAVES) {
            const float2 t = a.part_ml[slot(i)];
            weight[i] = t.x;
            m = fmaxf(m, t.x);
            if (i < 64 * WAVES) l = t.y;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, st::xor_lane(m, o, lane));
        if constexpr (WAVES > 1) {
            if (lane == 0) stat[wave] = m;
            __syncthreads();
            m = fmaxf(fmaxf(stat[0], stat[1]), fmaxf(stat[2], stat[3]));
        }
        m += ROOM;
        float sum = 0.f;
        for (int i = me; i < parts; i += 64 * WAVES) {
            const float w = weight[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(weight[i] - m);  // a power of two
            weight[i] = w;
            sum += w * (i < 64 * WAVES ? l : a.part_ml[slot(i)].y);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += st::xor_lane(sum, o, lane);
        if constexpr (WAVES > 1) {
            if (lane == 0) stat[4 + wave] = sum;
            __syncthreads();
            sum = (stat[4] + stat[5]) + (stat[6] + stat[7]);
        }
        if (gr < GROUPS) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int i0 = gr; i0 < parts; i0 += 8 * GROUPS) {
                if (i0 > gr) load(i0);
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float w = i0 + k * GROUPS < parts ? weight[i0 + k * GROUPS] : 0.f;
                    if (w != 0.f) v.x += w * x[k].x, v.y += w * x[k].y, v.z += w * x[k].z, v.w += w * x[k].w;
                }
            }
            *(float4 *)&red[team][gr][e] = v;
        }
        if constexpr (WAVES > 1) __syncthreads();
        const Ending ending(a, m, sum);
        const int token = (int)(((float)(joint.head % a.share + y) + 0.5f) * a.inv_share);
        const int64_t row = (int64_t)(joint.token + token) * a.hq + joint.head + y - token * a.share;
        for (int d = me; d < HD; d += 64 * WAVES) {
            float v = 0.f;
#pragma unroll
            for (int i = 0; i < GROUPS; i++) v += red[team][i][d];
            v = ending(v);
            const int64_t to = row * HD + d;
            if (a.dtype == ST_F32)
                ((float *)a.out)[to] = v;
            else if (a.dtype == ST_F16)
                ((_Float16 *)a.out)[to] = (_Float16)v;
            else
                ((__bf16 *)a.out)[to] = (__bf16)v;
        }
        if (a.lse && me == 0) a.lse[row] = ending.lse;
        if constexpr (WAVES > 1) __syncthreads();  // a row's values are read before the next one's are written
    }
}

// How a call is cut: rows of a tile (64 rt), workgroups, rows of a slot for parts of units (0: none is shared), rows of a unit on
// average, and whether a unit is of many workgroups.
struct Cut {
    int rows, rt, groups, part_rows, usual;
    bool many_parts;
};

Cut cut_of(int32_t dtype, int64_t n, int64_t nseq, int64_t hq, int64_t hkv, int64_t hd, int64_t max_pages, int64_t page) {
    Cut c;
    const int64_t rows = n * (hq / hkv);
    // 32 rows a wave share the work of taking codes apart, but keep two waves to a SIMD and not three: sequences of 16 rows on
    // average take 95 us with 16 and 112 with 32 a wave, of 64 rows 265 and 195.
    c.rt = hd <= 128 && rows >= 64 * nseq ? 2 : 1, c.rows = 64 * c.rt;
    const int per_cu = c.rt == 1 && hd <= 128 ? 3 : 2;
    c.groups = std::min(per_cu * st::device_cus(), MAX_GROUPS) & ~7;
    c.part_rows = max_pages * page <= WHOLE ? 0 : (int)std::min<int64_t>(c.rows, rows);
    c.usual = (int)std::min<int64_t>((rows + nseq - 1) / nseq, c.part_rows);
    c.many_parts = c.groups >= 32 * hkv * std::max(nseq, rows / c.rows);
    return c;
}

int64_t work_of(const Cut &c, int64_t hd) { return c.part_rows ? (int64_t)2 * c.groups * c.part_rows * (hd + 2) * 4 + c.groups * sizeof(Joint) : 0; }

}  // namespace

extern "C" int64_t st_kv_attention_4bit_bytes(int32_t dtype, int64_t n, int64_t nseq, int64_t hq, int64_t hkv, int64_t hd,
                                              int64_t max_pages, int64_t page) {
    if (n <= 0 || nseq <= 0 || hkv <= 0 || hq < hkv || max_pages <= 0) return 0;
    return work_of(cut_of(dtype, n, nseq, hq, hkv, hd, max_pages, page), hd);
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
    if (n < 0 || n > MAX_ROWS / hq)
        return st::fail(ST_ERR_INVALID, "%s: %lld rows of %lld heads (up to 2^26 in all)",
                        name, (long long)n, (long long)hq);
    if (dtype < ST_F32 || dtype > ST_BF16)
        return st::fail(ST_ERR_INVALID, "%s: dtype %d is none of ST_F32, ST_F16, ST_BF16",
                        name, (int)dtype);
    if (q_stride < hq * hd)
        return st::fail(ST_ERR_INVALID, "%s: rows of %lld elements lie %lld apart",
                        name, (long long)(hq * hd), (long long)q_stride);
    if (window < 0 || (window > 0 && !causal))
        return st::fail(ST_ERR_INVALID, "%s: a window of %lld keys%s",
                        name, (long long)window, causal ? "" : " without the causal mask");
    AttnArgs a = {};
    if (!st::cache_ok(name, a.c, nseq, table, max_pages, pages, page, hkv, k_codes, k_scales, v_codes, v_scales)) return ST_ERR_INVALID;
    if (n == 0 || nseq == 0) return ST_OK;
    if (!q || !q_start || !kv_len || !out) return st::fail(ST_ERR_INVALID, "%s: NULL buffer", name);
    const int64_t size = st::dtype_size(dtype);
    if (((uintptr_t)q | (uintptr_t)out) & (size - 1))
        return st::fail(ST_ERR_INVALID, "%s: q or out not aligned to its elements",
                        name);
    const Cut cut = cut_of(dtype, n, nseq, hq, hkv, hd, max_pages, page);
    if (cut.part_rows > 0 && (!work || ((uintptr_t)work & 15) || work_bytes < work_of(cut, hd)))
        return st::fail(ST_ERR_INVALID, "%s: work is %lld bytes of 16-byte aligned device memory, got %lld", name,
                        (long long)work_of(cut, hd), (long long)(work ? work_bytes : 0));
    if (!st::device_ok()) return ST_ERR_NO_DEVICE;
    a.q = q, a.out = out, a.lse = lse, a.q_start = q_start, a.kv_len = kv_len;
    a.part_o = (float *)work, a.part_ml = (float2 *)((float *)work + (int64_t)2 * cut.groups * cut.part_rows * hd);
    a.joints = (Joint *)(a.part_ml + (int64_t)2 * cut.groups * cut.part_rows);
    a.q_stride = q_stride;
    a.scale2 = scale * 1.44269504088896341f;
    a.n = (int32_t)n, a.hq = (int32_t)hq, a.dtype = dtype, a.causal = causal != 0, a.one = one != 0;
    a.window = window > INT32_MAX / 2 ? 0 : (int32_t)window;
    a.groups = cut.groups, a.part_rows = cut.part_rows;
    a.share = (int32_t)(hq / hkv), a.cap = (int32_t)(max_pages * page);
    a.per = a.share <= cut.rows ? cut.rows / a.share : 0;
    a.tile_rows = a.per ? a.per * a.share : cut.rows;
    const int64_t room = std::max(a.cap, 1);
    a.most = (int32_t)(a.window > 0 ? std::min<int64_t>(room, (int64_t)a.window + std::max(a.per, 1) + 63) : room);
    a.lead = LEAD;
    a.small = nseq <= 64 && (room + a.tile_rows + a.lead) * hkv * nseq < INT32_MAX;
    a.inv_share = 1.f / (float)a.share, a.inv_groups = 1.f / (float)cut.groups;
    a.vec_q = st::rows_aligned(q, q_stride, size), a.vec_out = ((uintptr_t)out & 15) == 0;
    auto go = [&](auto hd_) -> st_status {
        constexpr int HD = decltype(hd_)::value;
        const hipStream_t s = st::stream_of(stream);
        const uint32_t grid = cut.groups;
        auto with = [&](auto f32, auto f16, auto bf16) { (dtype == ST_F32 ? f32 : dtype == ST_F16 ? f16 : bf16)<<<grid, 256, 0, s>>>(a); };
        // f16 outputs show the rounding of the weights to f16 (1.4 times the error of their own rounding).  Two parts cost few rows
        // little (64 sequences 88.1 and 88.7 us, one long one 46.6 and 48.1), a prompt 529 and 579: there one does.  Which it is
        // goes by the batch (cut_of), so a single f16 token beside a long prompt may have its weights in one part too.  bf16
        // outputs are rounded eight times coarser and hardly show it (1.74e-3 to 1.76e-3 off): one part always.
        if (cut.rt == 1)
            with(k_attention4<HD, 2, 2, 1>, k_attention4<HD, 1, 2, 1>, k_attention4<HD, 1, 1, 1>);
        else if constexpr (HD <= 128)
            with(k_attention4<HD, 2, 2, 2>, k_attention4<HD, 1, 1, 2>, k_attention4<HD, 1, 1, 2>);
        ST_LAUNCH_CHECK();
        if (cut.part_rows == 0) return ST_OK;
        // Four waves a row where it has many parts (one long sequence: 45.7 us with four, 49.7 with one),
        // else one (64 sequences: 88.8, 86.1; a prompt of 2048 tokens: 592, 531).
        if (cut.many_parts)
            k_merge4<HD, 4><<<dim3(grid, cut.usual), 256, 0, s>>>(a);
        else
            k_merge4<HD, 1><<<dim3(grid, (cut.usual + 3) / 4), 256, 0, s>>>(a);
        ST_LAUNCH_CHECK();
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
