// Products of 8-bit rows and 8-bit weights (quant8.h): out[i, j] = (sum over l of x[i, l] w[j, l]) xs[i] ws[j] + bias[j], then
// ReLU; and the gated form act(gate) up of two such products.  Sums of codes are exact in 32-bit integers (k <= 131072; 2^31 is
// reached by 131072 products of -128 and -128 alone, a code that the format does not have); the scales enter once, in f32.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.h"
#include "dma_tile.h"
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

// act(g) u.  silu is g / (1 + exp(-g)).  gelu is g Phi(g) = g erfc(-g / sqrt 2) / 2, with erfc(z) = exp(-z^2) t P(t), t = 1 / (1 + z / 2),
// for z >= 0: P of degree 8, its numbers as f32 holds them, is within 4.6e-8 of erfc for all z up to 14 (least squares of the relative error,
// one number after the other rounded and the rest fitted anew; erfc(14) is 0 in f32), and the tail stays where 1 + erf would
// cancel.  Measured, relative: gelu is off by up to 4e-7 for |g| < 1 (the reciprocal's last place, by which t is off), 1.2e-7 above, 8e-7 down to
// g = -4, 3e-6 to -8, 8e-6 to -13 (the exponent's rounding); silu by 1.8e-7 for g > -1, 5e-7 to -8, 4e-6 to -80.  About 20
// operations; the library's erfcf takes some 100.
__device__ __forceinline__ float gated(float g, float u, int32_t act) {
    if (act == ST_ACT_SILU) return g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * g)) * u;
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.35355339f, __builtin_fabsf(g), 1.f));
    float p = -0.059389167f;
    p = __builtin_fmaf(p, t, 0.28613672f);
    p = __builtin_fmaf(p, t, -0.49043193f);
    p = __builtin_fmaf(p, t, 0.2817614f);
    p = __builtin_fmaf(p, t, -0.02916681f);
    p = __builtin_fmaf(p, t, 0.20375963f);
    p = __builtin_fmaf(p, t, 0.24283351f);
    p = __builtin_fmaf(p, t, 0.2824123f);
    p = __builtin_fmaf(p, t, 0.28208432f);
    const float half = 0.5f * p * (t * __builtin_amdgcn_exp2f(-0.72134752f * g * g));  // Phi(-|g|)
    return g * (g < 0.f ? half : 1.f - half) * u;
}

// sum xs ws + bias.  A sum is below 2^31, so it can be multiplied by the row's scale first up to 2^96; a larger one comes last, and the sum
// times the channel's passes f32's range only where the result does too.  (A sum times a subnormal scale loses nothing.)
__device__ __forceinline__ float scaled(int32_t sum, float xs, float ws, float bias) {
    const bool last = __builtin_fabsf(xs) >= 0x1p96f;
    return __builtin_fmaf((float)sum * (last ? ws : xs), last ? xs : ws, bias);
}

// 16 codes from p on, of which `left` are inside the row; unaligned rows are read a byte at a time.
__device__ __forceinline__ i4 load16(const int8_t *p, int64_t left, bool vec) {
    uint32_t v[4] = {0, 0, 0, 0};
    if (vec && left >= 16) return *(const i4 *)p;
#pragma unroll
    for (int i = 0; i < 16; i++)
        if (i < left) v[i >> 2] |= (uint32_t)(uint8_t)p[i] << (8 * (i & 3));
    return i4{(int)v[0], (int)v[1], (int)v[2], (int)v[3]};
}

// Any strides and alignment, and offsets past a tile's 32 bits: 64 rows of x by 64 rows of weights a workgroup, 32 x 32 a wave; a gated
// product's 64 are 32 of the gate's and the same 32 of the other half's.
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

// Rows from `p` on as a buffer of `bytes` (up to 4 GB), whose loads give 0 past the end.  It begins 4 KB before p: offsets into it are
// 4096 and more, as the loads' own offsets count both there and in LDS.
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u4 rows_at(const int8_t *p, int64_t bytes) {
    const uint64_t base = (uint64_t)p - 4096;
    return u4{st::lane_value((uint32_t)base, 0), st::lane_value((uint32_t)(base >> 32) & 0xFFFF, 0),
              st::lane_value((uint32_t)min(bytes + 4096, (int64_t)0xFFFFFFFF), 0), 0x00020000};
}

// L 16-byte loads a lane (1 KB a wave each), one behind the other in LDS from `to` on: lane l's of load i lands at to + 1024 i + 16 l
// and comes from offset off[i] + 1024 i + along.  ONCE: rows that nobody else reads pass by the L2 (nontemporal).
template <int L, bool ONCE>
__device__ __forceinline__ void dma_rows(u4 rows, const uint32_t *off, uint32_t along, uint32_t to) {
    static_assert(L == 1 || L == 2, "loads at once");
    uint32_t saved;
#define ST_DMA2(NT)                                                                                                                    \
    asm volatile(                                                                                                                      \
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\t"                                                                          \
        "buffer_load_dwordx4 %1, %4, %5 offen" NT " lds\n\tbuffer_load_dwordx4 %2, %4, %5 offen offset:1024" NT " lds\n\t"            \
        "s_mov_b32 m0, %0"                                                                                                             \
        : "=&s"(saved) : "v"(off[0]), "v"(off[1]), "s"(to), "s"(rows), "s"(along) : "memory")
#define ST_DMA1(NT)                                                                                                                    \
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %3, %4 offen" NT " lds\n\ts_mov_b32 m0, %0" \
                 : "=&s"(saved) : "v"(off[0]), "s"(to), "s"(rows), "s"(along) : "memory")
    if constexpr (L == 2 && ONCE)
        ST_DMA2(" nt");
    else if constexpr (L == 2)
        ST_DMA2("");
    else if constexpr (ONCE)
        ST_DMA1(" nt");
    else
        ST_DMA1("");
#undef ST_DMA2
#undef ST_DMA1
}

// A word a lane: lane l's comes from p and lands at to + 4 l.
__device__ __forceinline__ void dma_words(const void *p, uint32_t to) {
    uint32_t saved;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(saved) : "v"(p), "s"(to) : "memory");
}

// The place of unit `at` among tiles: they go down GROUP rows of tiles, then one to the right, so that neighbours share panels.
struct Tile {
    int m, n;
    __device__ __forceinline__ Tile(uint32_t at, uint32_t tiles_m, uint32_t tiles_n) {
        constexpr uint32_t GROUP = 8;
        const uint32_t first = at / (GROUP * tiles_n) * GROUP, high = min(GROUP, tiles_m - first), in = at - first * tiles_n;
        m = (int)(first + in % high), n = (int)(in / high);
    }
};

// Workgroups go to the 8 XCDs in turn.  Each XCD has a run of the units, whose panels its L2 then holds, and its workgroups take them in
// turn: the first one's place, the step, and the run's end.
struct Run {
    uint32_t first, step, end;
    __device__ __forceinline__ Run(uint32_t id, uint32_t groups, uint32_t total) {
        const uint32_t xcd = id % 8, start = xcd * (total / 8) + min(xcd, total % 8);
        first = start + id / 8, step = (groups - xcd + 7) / 8, end = start + total / 8 + (xcd < total % 8);
    }
};

struct Units {
    uint32_t tiles_m, tiles_n, slices, total;  // total = tiles_m tiles_n slices
    int32_t slice;                             // stages of a slice
};

template <int BK>
__device__ __forceinline__ int swizzle(int r) { return BK == 64 ? (r >> 2) & 3 : BK == 128 ? (r >> 1) & 7 : r & 15; }

constexpr int STAGED = 128 + 16;  // bytes of a staged row of out

// A kernel's tile: rows of x and of weights (four waves, two down and two across), k of a stage, stages in LDS.  ONCE: there is one tile
// of rows of x, so that the weights are read once.
template <int BM_, int BN_, int BK_, int NS_, bool ONCE_ = false>
struct Shape {
    static constexpr bool ONCE = ONCE_;
    static constexpr int BM = BM_, BN = BN_, DOWN = 2, ACROSS = 2, BK = BK_, NS = NS_, WM = BM / DOWN, WN = BN / ACROSS;
    static constexpr int XS = std::max(WM, 64), WS = std::max(WN, 64);  // words of a wave's tables (the DMA brings 64 at once)
    static constexpr int LDS = NS * (BM + BN) * BK + 4 * (32 * STAGED + (XS + 2 * WS) * 4);
    static constexpr int AT_ONCE = 160 * 1024 / LDS;  // workgroups of a CU (as LDS goes)
};

// Tiles of BM rows of x by BN rows of weights, four waves, k in stages of BK bytes that the LDS DMA brings,
// NS of them in LDS.  Products are 32x32x32 with the weights as the first operand, so that a lane's sums are of one row of x and
// runs of four columns.  T int32_t: sums of a slice of k, [slices, m, n], for k_join8.
//
// LDS: [row][BK / 16 chunks of 16 k]; chunk c of row r is in slot c ^ swizzle(r), so that the 16 rows a quarter of a wave reads
// are in 16 different groups of four banks.  A wave reads the fragments of the next 32 k while it multiplies these; with a
// stage's last 32 k in registers its slot is free, so behind the barrier that says so of all waves (and that the next stage has landed)
// the stage NS further on is on its way into it.
//
// A workgroup stays and takes a unit (a tile, or a slice of its k) after another: the stages of all its units are one stream, and the next
// unit's first are in flight while one's sums are scaled and stored.
//
// A gated tile's rows of weights are, 32 by 32 in turn, the gate's and the other half's of the same columns, so that a wave holds both
// sums of an output.  Rows past the end repeat the last one and are not stored; x's bytes past k are zeros in LDS.
//
// 8192 x 8192 x 8192 to bf16: 445 to 480 us on several cards, 2,290 to 2,470 TOP/s, bound by the card's power (operands of zeros:
// 3,140); 4095 x 4096 x 2 x 12288 with gelu 402 to 410 us; a tile's outputs take 8 us in which its products wait.  48 x 4096 x 11003 in tiles
// of 64 x 64: 14 us, 172 workgroups.
template <class T, bool GATED, class Tiles>
__global__ __launch_bounds__(256, std::min(Tiles::AT_ONCE, 4)) void k_product8(Product a, Units units) {
    constexpr int BM = Tiles::BM, BN = Tiles::BN, BK = Tiles::BK, NS = Tiles::NS, WM = Tiles::WM, WN = Tiles::WN, XS = Tiles::XS, WS = Tiles::WS;
    constexpr bool PART = std::is_same_v<T, int32_t>;
    constexpr int C = BK / 16, PER = 64 / C, LX = BM / (4 * PER), LW = BN / (4 * PER), SX = BM * BK, SW = BN * BK, KS = BK / 32, S = LX < 2 || LW < 2 ? 1 : 2;
    constexpr int FM = WM / 32, FN = WN / 32, BOTH = GATED ? 2 : 1;
    constexpr int COLUMNS = BN / BOTH, WCOLS = WN / BOTH;  // of out: a tile's, a wave's
    constexpr int STORES = WM * WCOLS * (int)sizeof(T) / 1024;  // of a wave and unit
    static_assert(KS % 2 == 0 && FN % BOTH == 0 && !(PART && GATED), "fragments in pairs");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / Tiles::ACROSS, wn = wave % Tiles::ACROSS;
    const uint32_t ring = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char *)lds;
    char *const staged = lds + NS * (SX + SW) + wave * 32 * STAGED;
    float *const table = (float *)(lds + NS * (SX + SW) + 4 * 32 * STAGED) + wave * (XS + 2 * WS);  // xs, ws and bias of this wave
    const int all = (int)((a.k + BK - 1) / BK), left = (int)(a.k - (int64_t)(all - 1) * BK);  // stages; bytes of a row in the last one
    const int64_t whole_k = (a.k + 15) & ~(int64_t)15;  // (rows are read in whole units)
    const Run run(blockIdx.x, gridDim.x, units.total);

    // What is being brought: a unit's stages, from those of the unit `coming` on.
    uint32_t coming = run.first;
    int st_in = 0, end_in = 0;
    u4 xrows, wrows;
    uint32_t xo[LX], wo[LW];
    auto slice_of = [&](uint32_t unit, int &from, int &to) {
        const int s = (int)(unit % units.slices);
        from = s * units.slice, to = min(from + units.slice, all);
    };
    auto next_unit = [&] {
        const Tile tile(coming / units.slices, units.tiles_m, units.tiles_n);
        slice_of(coming, st_in, end_in);
        const int64_t m0 = (int64_t)tile.m * BM, n0 = (int64_t)tile.n * COLUMNS;
        xrows = rows_at(a.x + m0 * a.x_stride, (a.m - 1 - m0) * a.x_stride + whole_k);
        wrows = rows_at(a.w + n0 * a.w_stride, ((GATED ? 2 * a.n : a.n) - 1 - n0) * a.w_stride + whole_k);
#pragma unroll
        for (int i = 0; i < LX; i++) {
            const int p = (wave * LX + i) * 64 + lane, r = p / C, c = (p % C) ^ swizzle<BK>(r);
            xo[i] = (uint32_t)min((int64_t)r, a.m - 1 - m0) * (uint32_t)a.x_stride + c * 16 + 4096 - 1024 * (i % S);
        }
#pragma unroll
        for (int i = 0; i < LW; i++) {
            const int p = (wave * LW + i) * 64 + lane, r = p / C, c = (p % C) ^ swizzle<BK>(r);
            const uint32_t row = GATED ? (uint32_t)min((int64_t)(r / 64 * 32 + r % 32), a.n - 1 - n0) + (r / 32 % 2) * (uint32_t)a.n
                                       : (uint32_t)min((int64_t)r, a.n - 1 - n0);
            wo[i] = row * (uint32_t)a.w_stride + c * 16 + 4096 - 1024 * (i % S);
        }
    };
    // Load l, S at once, of the stage that comes next.
    auto bring = [&](int l, uint32_t to) {
        if (l < LX / S)
            dma_rows<S, false>(xrows, xo + l * S, (uint32_t)st_in * BK, to + (wave * LX + l * S) * 1024);
        else
            dma_rows<S, Tiles::ONCE>(wrows, wo + (l * S - LX), (uint32_t)st_in * BK, to + SX + (wave * LW + l * S - LX) * 1024);
    };
    // The stage after it.  Behind the last unit's last stage that one comes again (and is not used), so that there are always as many
    // on their way.
    auto brought = [&] {
        if (st_in + 1 < end_in) {
            st_in++;
        } else if (coming + run.step < run.end) {
            coming += run.step;
            next_unit();
        }
    };

    int at[KS];  // this lane's bytes of a block of 32 rows, for each 32 k
#pragma unroll
    for (int s = 0; s < KS; s++) at[s] = (lane & 31) * BK + (((2 * s + (lane >> 5)) ^ swizzle<BK>(lane & 31)) * 16);
    // Fragments of a k step, in the order of their use: the weights' first block's, x's, the weights' others.
    i4 f[2][FN + FM];
    auto piece = [&](uint32_t slot, int s, int q, i4 *into) {
        const char *const x = lds + slot + wm * WM * BK + at[s], *const w = lds + slot + SX + wn * WN * BK + at[s];
        if (q == 0 || q > FM)
            into[q ? q - FM : 0] = *(const i4 *)(w + (q ? q - FM : 0) * 32 * BK);
        else
            into[FN + q - 1] = *(const i4 *)(x + (q - 1) * 32 * BK);
    };
    // x's bytes past k, in a row's last stage, which has landed everywhere: zeros.
    auto end_rows = [&](uint32_t g) {
        char *const x = lds + g % NS * (SX + SW);
        for (int u = tid; u < BM * C; u += 256) {
            const int r = u / C, c = u % C;
            char *const p = x + r * BK + ((c ^ swizzle<BK>(r)) * 16);
            if (16 * c >= left)
                *(i4 *)p = i4{0, 0, 0, 0};
            else if (16 * c + 16 > left)
                for (int b = left - 16 * c; b < 16; b++) p[b] = 0;
        }
        dma::bar_written();
    };

    if constexpr (!PART) {
        if (!a.bias)
            for (int i = lane; i < WS; i += 64) table[XS + WS + i] = 0.f;
    }
    next_unit();
    for (int i = 0; i < NS; i++) {
#pragma unroll
        for (int l = 0; l < (LX + LW) / S; l++) bring(l, ring + i * (SX + SW));
        brought();
    }
    dma::wait_vm<(NS - 1) * (LX + LW)>();
    dma::bar_written();
    {
        int from, to;
        slice_of(run.first, from, to);
        if (from == all - 1 && left < BK) end_rows(0);
    }
#pragma unroll
    for (int q = 0; q < FN + FM; q++) piece(0, 0, q, f[0]);

    uint32_t g = 0;       // the stage that is multiplied, of this workgroup's
    int older = 0;        // coming stages that were on their way before the last unit's STORES stores of this wave
    for (uint32_t unit = run.first; unit < run.end; unit += run.step) {
        const Tile tile(unit / units.slices, units.tiles_m, units.tiles_n);
        const int64_t row0 = (int64_t)tile.m * BM + wm * WM, col0 = (int64_t)tile.n * COLUMNS + wn * WCOLS;  // of this wave
        int from, to;
        slice_of(unit, from, to);
        if constexpr (!PART) {  // the wave's scales and bias, for when the sums are there
            const uint32_t where = ring + (uint32_t)((char *)table - lds);
#pragma unroll
            for (int i = 0; i < (WM + 63) / 64; i++) dma_words(a.xs + min(row0 + min(64 * i + lane, WM - 1), a.m - 1), where + 256 * i);
#pragma unroll
            for (int i = 0; i < (WN + 63) / 64; i++) {
                const int r = min(64 * i + lane, WN - 1);
                const int64_t row = GATED ? min(col0 + r / 64 * 32 + r % 32, a.n - 1) + (r / 32 % 2) * a.n : min(col0 + r, a.n - 1);
                dma_words(a.ws + row, where + 4 * XS + 256 * i);
                if (a.bias) dma_words(a.bias + row, where + 4 * (XS + WS) + 256 * i);
            }
        }
        i16 acc[FN][FM];
        i4 zero = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < FN; j++)
#pragma unroll
            for (int i = 0; i < FM; i++) {  // zeros by products of zeros, 32 cycles for 16 registers (which are as many writes otherwise)
                asm volatile("" : "+v"(zero));  // (another one each time: the compiler would copy one result)
                acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(zero, zero, i16{}, 0, 0, 0);
            }
        // Every operation of a stage stands between two products: the compiler's own order leaves the matrix cores waiting for the
        // barrier, the loads' addresses and the fragments in turn (8192 x 16384 x 8192 in stages of 64 k: 2,060 TOP/s so, 2,270 in this order).
        for (int st = from; st < to; st++) {
            constexpr int N = FM * FN, PIECES = FN + FM, LOADS = (LX + LW) / S, MOVES = N > 8 ? N - 4 : N - 1;
            static_assert(std::min(N - 1, 2 + (LOADS - 1) * (5 * N / 8) / LOADS) <= MOVES, "all of a stage's loads before the next stage's place");
            const uint32_t slot = g % NS * (SX + SW), next = (g + 1) % NS * (SX + SW);
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int n = 0; n < N; n++) {
                    acc[n / FM][n % FM] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f[s & 1][n / FM], f[s & 1][FN + n % FM], acc[n / FM][n % FM], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                    if (s < KS - 1) {
#pragma unroll
                        for (int q = 0; q < PIECES; q++)
                            if (n == q * (3 * N / 4) / PIECES) piece(slot, s + 1, q, f[(s + 1) & 1]);
                    } else {
                        if (n == 0) {
                            // The next stage has landed.  (The stages on their way when the last unit's outputs were stored are older
                            // than those stores, and need not wait for them.)
                            if (older > 0) {
                                dma::wait_vm<std::min((NS - 2) * (LX + LW) + STORES, 63)>();
                                older--;
                            } else {
                                dma::wait_vm<(NS - 2) * (LX + LW)>();
                            }
                            dma::bar_written();  // (and this one's fragments are read)
                            if (left < BK) {
                                int after = st + 1, end;
                                if (after == to) slice_of(unit + run.step, after, end);
                                if (after == all - 1) end_rows(g + 1);
                            }
                        }
#pragma unroll
                        for (int q = 0; q < PIECES; q++)
                            if (n == std::min(N - 1, 1 + q * (3 * N / 4) / PIECES)) piece(next, 0, q, f[0]);
#pragma unroll
                        for (int l = 0; l < LOADS; l++)
                            if (n == std::min(N - 1, 2 + l * (5 * N / 8) / LOADS)) bring(l, ring + slot);
                        if (n == MOVES) brought();
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            g++;
        }

        // 32 rows of x and 128 bytes of columns at a time: scaled and rounded, through this wave's part of LDS, whole 128-byte runs
        // of rows to memory.
        if (!PART && to - from <= NS) dma::wait_vm<0>();  // (else the table is behind stages that have been waited for)
        asm volatile("" ::: "memory");
        T *const out = PART ? (T *)a.out + (int64_t)(unit % units.slices) * a.m * a.n : (T *)a.out;  // (slices of sums)
        const int64_t stride = PART ? a.n : a.out_stride;
        constexpr int V = 16 / (int)sizeof(T), BLOCKS = std::min(128 / (int)sizeof(T), WCOLS) / 32;
        typedef T T4 __attribute__((ext_vector_type(4)));
        typedef float F4 __attribute__((ext_vector_type(4)));
        typedef T TV __attribute__((ext_vector_type(V)));
        // A sum out of the matrix cores' registers, when it is wanted (the compiler would move all of them at once, and put others away).
        auto sum_of = [&](int j, int i, int e) {
            int32_t v;
            asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(acc[j][i][e]));
            return v;
        };
        asm volatile("s_nop 15\n\ts_nop 15");  // the last product's results are there
        typedef T TU __attribute__((ext_vector_type(V), aligned(sizeof(T))));
        const bool whole = row0 + WM <= a.m && col0 + WCOLS <= a.n;
        older = whole ? NS - 1 : 0;
#pragma unroll
        for (int b = 0; b < WCOLS / 32; b += BLOCKS) {
            F4 ws[BLOCKS * BOTH][4], bias[BLOCKS * BOTH][4];
            if constexpr (!PART) {
#pragma unroll
                for (int h = 0; h < BLOCKS * BOTH; h++)
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const int c = (b * BOTH + h) * 32 + 8 * q + 4 * (lane >> 5);
                        ws[h][q] = *(const F4 *)(table + XS + c), bias[h][q] = *(const F4 *)(table + XS + WS + c);
                    }
            }
#pragma unroll
            for (int i = 0; i < FM; i++) {
                const float xs = PART ? 0.f : table[i * 32 + (lane & 31)];
#pragma unroll
                for (int h = 0; h < BLOCKS; h++)
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        T4 v;
                        if constexpr (PART) {
#pragma unroll
                            for (int e = 0; e < 4; e++) v[e] = sum_of((b + h) * BOTH, i, 4 * q + e);
                        } else {
                            F4 y;
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                y[e] = scaled(sum_of((b + h) * BOTH, i, 4 * q + e), xs, ws[h * BOTH][q][e], bias[h * BOTH][q][e]);
                                if constexpr (GATED)
                                    y[e] = gated(y[e], scaled(sum_of((b + h) * BOTH + 1, i, 4 * q + e), xs, ws[h * BOTH + 1][q][e], bias[h * BOTH + 1][q][e]), a.act);
                            }
                            if (!GATED && a.act == ST_ACT_RELU) {
                                asm volatile("");  // (a branch, not selects)
#pragma unroll
                                for (int e = 0; e < 4; e++) y[e] = y[e] < 0.f ? 0.f : y[e];
                            }
                            v = __builtin_convertvector(y, T4);
                        }
                        *(T4 *)(staged + (lane & 31) * STAGED + (h * 32 + 8 * q + 4 * (lane >> 5)) * (int)sizeof(T)) = v;
                    }
                constexpr int LINE = BLOCKS * 32 / V, AT_ONCE = 64 / LINE;  // lanes of a row, rows at once
                const int c = lane % LINE * V;
                const uint32_t mine = (uint32_t)(lane / LINE * stride + c) * (uint32_t)sizeof(T);  // (rows of out are less than 2^23 bytes apart)
                char *o = (char *)(out + (row0 + i * 32) * stride + col0 + b * 32);
#pragma unroll
                for (int r0 = 0; r0 < 32; r0 += AT_ONCE, o += AT_ONCE * stride * (int64_t)sizeof(T)) {
                    const TV v = *(const TV *)(staged + (r0 + lane / LINE) * STAGED + c * (int)sizeof(T));
                    if (whole && BM == 256) {  // (large outputs leave the L2 to the operands: 8192 x 8192 x 8192 457 us, 460 otherwise)
                        __builtin_nontemporal_store(*(const TU *)&v, (TU *)(o + mine));
                    } else if (whole) {
                        *(TU *)(o + mine) = v;
                    } else if (row0 + i * 32 + r0 + lane / LINE < a.m) {
                        const int64_t n = a.n - col0 - b * 32 - c;  // columns from here on
                        if (n >= V) {
                            *(TU *)(o + mine) = v;
                        } else {
#pragma unroll
                            for (int e = 0; e < V; e++)
                                if (e < n) ((T *)(o + mine))[e] = v[e];
                        }
                    }
                }
            }
        }
    }
    dma::wait_vm<0>();  // (no stage may land after the workgroup has left its LDS to another)
}

// A few rows of x, 16 MB of them, by 16 NT rows of weights a workgroup, whose waves share k.  Bound by the weights' bytes: a lane
// reads 32 of one row (a load is 64 bytes of each of 16 rows, two loads whole lines), straight into the registers that
// 16x16x64 products take, U steps of 128 k at once; nothing goes through LDS but the waves' sums at the end.  (These products run
// at half the rate of 32x32x32, which does not show: 5 TB/s of weights keep a SIMD busy one cycle in 13 MB at 16 rows.)
// A gated product's NT is 2: the gate's rows and the other half's of the same columns.
template <class T, bool GATED, int MB, int NT, int WAVES, int U>
__global__ __launch_bounds__(64 * WAVES) void k_few8(Product a) {
    constexpr int BOTH = GATED ? 2 : 1, COLUMNS = 16 * NT / BOTH, PITCH = 16 * NT + 4;
    static_assert(!GATED || NT == 2, "both halves");
    __shared__ __attribute__((aligned(16))) int32_t sums[WAVES][16 * MB][PITCH];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, q = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * COLUMNS, m0 = (int64_t)blockIdx.y * 16 * MB;
    const int8_t *w[NT], *x[MB];
#pragma unroll
    for (int t = 0; t < NT; t++) w[t] = a.w + (GATED ? min(n0 + i, a.n - 1) + t * a.n : min(n0 + 16 * t + i, a.n - 1)) * a.w_stride + 32 * q;
#pragma unroll
    for (int b = 0; b < MB; b++) x[b] = a.x + min(m0 + 16 * b + i, a.m - 1) * a.x_stride + 32 * q;
    i4 acc[NT][MB];
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int b = 0; b < MB; b++) acc[t][b] = i4{0, 0, 0, 0};
    const int full = (int)(a.k / 128);
    auto steps = [&](int from, auto count_) {  // `from` and every WAVES-th after it
        constexpr int COUNT = decltype(count_)::value;
        i4 wf[COUNT][NT][2], xf[COUNT][MB][2];
#pragma unroll
        for (int u = 0; u < COUNT; u++) {
            const int64_t at = (int64_t)(from + u * WAVES) * 128;
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int t = 0; t < NT; t++) wf[u][t][h] = __builtin_nontemporal_load((const i4 *)(w[t] + at + 16 * h));
#pragma unroll
                for (int b = 0; b < MB; b++) xf[u][b][h] = *(const i4 *)(x[b] + at + 16 * h);
            }
        }
#pragma unroll
        for (int u = 0; u < COUNT; u++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int b = 0; b < MB; b++) acc[t][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u][t][h], xf[u][b][h], acc[t][b], 0, 0, 0);
    };
    int s = wave;
    for (; s + (U - 1) * WAVES < full; s += U * WAVES) steps(s, std::integral_constant<int, U>());
    for (; s < full; s += WAVES) steps(s, std::integral_constant<int, 1>());
    if (s == full && a.k % 128) {  // the part of a step behind the last: x's codes past k are zeros, units past k are not read
        const int64_t at = (int64_t)full * 128;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int left = (int)(a.k - at) - 32 * q - 16 * h;
            i4 wf[NT], xf[MB];
#pragma unroll
            for (int t = 0; t < NT; t++) wf[t] = left > 0 ? *(const i4 *)(w[t] + at + 16 * h) : i4{0, 0, 0, 0};
#pragma unroll
            for (int b = 0; b < MB; b++) {
                xf[b] = left > 0 ? *(const i4 *)(x[b] + at + 16 * h) : i4{0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int bytes = left - 4 * e;
                    if (bytes < 4) xf[b][e] = bytes > 0 ? xf[b][e] & ((1 << (8 * bytes)) - 1) : 0;
                }
            }
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int b = 0; b < MB; b++) acc[t][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[t], xf[b], acc[t][b], 0, 0, 0);
        }
    }
    // Lane (i, q) holds row i of x with rows 4 q .. 4 q + 3 of the weights.
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int b = 0; b < MB; b++) *(i4 *)&sums[wave][16 * b + i][16 * t + 4 * q] = acc[t][b];
    __syncthreads();
    for (int o = tid; o < 16 * MB * COLUMNS; o += 64 * WAVES) {
        const int b = o / COLUMNS, j = o % COLUMNS;
        const int64_t mi = m0 + b, ni = n0 + j;
        if (mi >= a.m || ni >= a.n) continue;
        int32_t sum = 0, other = 0;
#pragma unroll
        for (int v = 0; v < WAVES; v++) {
            sum += sums[v][b][j];
            if constexpr (GATED) other += sums[v][b][16 + j];
        }
        float y = scaled(sum, a.xs[mi], a.ws[ni], a.bias ? a.bias[ni] : 0.f);
        if constexpr (GATED)
            y = gated(y, scaled(other, a.xs[mi], a.ws[a.n + ni], a.bias ? a.bias[a.n + ni] : 0.f), a.act);
        else if (a.act == ST_ACT_RELU)
            y = y < 0.f ? 0.f : y;
        ((T *)a.out)[mi * a.out_stride + ni] = (T)y;
    }
}

// One to four rows of x: R rows of weights a wave, each read whole lines at a time (64 lanes by 16 bytes), U times 1024 k at once, and
// multiplied by four codes an instruction with x in LDS, which the workgroup's waves share; the lanes' sums are added up at the end.
// Streams of neighbouring lines are what a matrix operand's 64 bytes of 16 rows are not: one row through 32768 x 8192 39 us, 6.9 TB/s,
// bound by HBM (51 us with k_few8).
template <class T, bool GATED, int M, int R, int U>
__global__ __launch_bounds__(256) void k_one8(Product a) {
    constexpr int BOTH = GATED ? 2 : 1;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int chunks = (int)((a.k + 1023) / 1024), width = chunks * 1024, k = (int)a.k;
    for (int u = tid; u < M * (width / 16); u += 256) {
        const int m = u / (width / 16), at = u % (width / 16) * 16, left = k - at;
        i4 v = {0, 0, 0, 0};
        if (left > 0 && m < a.m) v = *(const i4 *)(a.x + m * a.x_stride + at);
        if (left < 16) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int bytes = left - 4 * e;
                if (bytes < 4) v[e] = bytes > 0 ? v[e] & ((1 << (8 * bytes)) - 1) : 0;
            }
        }
        *(i4 *)(lds + m * width + at) = v;
    }
    __syncthreads();
    for (int64_t n0 = ((int64_t)blockIdx.x * 4 + wave) * R; n0 < a.n; n0 += (int64_t)gridDim.x * 4 * R) {
        const int8_t *w[R * BOTH];
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int h = 0; h < BOTH; h++) w[r * BOTH + h] = a.w + (min(n0 + r, a.n - 1) + h * a.n) * a.w_stride;
        int32_t acc[R * BOTH][M];
#pragma unroll
        for (int r = 0; r < R * BOTH; r++)
#pragma unroll
            for (int m = 0; m < M; m++) acc[r][m] = 0;
        auto some = [&](int chunk, auto count_) {
            constexpr int COUNT = decltype(count_)::value;
            i4 v[COUNT][R * BOTH];
#pragma unroll
            for (int u = 0; u < COUNT; u++) {
                const int at = (chunk + u) * 1024 + lane * 16, from = at < k ? at : 0;  // (x is 0 past k)
#pragma unroll
                for (int r = 0; r < R * BOTH; r++) v[u][r] = __builtin_nontemporal_load((const i4 *)(w[r] + from));
            }
#pragma unroll
            for (int u = 0; u < COUNT; u++)
#pragma unroll
                for (int m = 0; m < M; m++) {
                    const i4 x = *(const i4 *)(lds + m * width + (chunk + u) * 1024 + lane * 16);
#pragma unroll
                    for (int r = 0; r < R * BOTH; r++)
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[r][m] = __builtin_amdgcn_sdot4(v[u][r][e], x[e], acc[r][m], false);
                }
        };
        int c = 0;
        for (; c + U <= chunks; c += U) some(c, std::integral_constant<int, U>());
        for (; c < chunks; c++) some(c, std::integral_constant<int, 1>());
        int32_t mine[BOTH] = {};
#pragma unroll
        for (int r = 0; r < R * BOTH; r++)
#pragma unroll
            for (int m = 0; m < M; m++) {
                int32_t v = acc[r][m];  // (step by step: a loop of six here stays a loop, 1 us a row of x)
                v += st::xor_lane(v, 32, lane), v += st::xor_lane(v, 16, lane), v += st::xor_lane(v, 8, lane);
                v += st::xor_lane(v, 4, lane), v += st::xor_lane(v, 2, lane), v += st::xor_lane(v, 1, lane);
                if (lane == r / BOTH * M + m) mine[r % BOTH] = v;
            }
        const int64_t m = lane % M, n = n0 + lane / M;
        if (lane >= R * M || m >= a.m || n >= a.n) continue;
        float y = scaled(mine[0], a.xs[m], a.ws[n], a.bias ? a.bias[n] : 0.f);
        if constexpr (GATED)
            y = gated(y, scaled(mine[BOTH - 1], a.xs[m], a.ws[a.n + n], a.bias ? a.bias[a.n + n] : 0.f), a.act);
        else if (a.act == ST_ACT_RELU)
            y = y < 0.f ? 0.f : y;
        ((T *)a.out)[m * a.out_stride + n] = (T)y;
    }
}

// out from the sums of slices of k, four columns a thread.  A gated product's sums are [slices, m, 2 n].  A launch's latency, 2 to 5 us: the
// sums are in the L2 (200 x 16384 x 512 14 us with its slices' product).
template <class T, bool GATED>
__global__ __launch_bounds__(256) void k_join8(Product a, const int32_t *__restrict__ part, int32_t slices) {
    typedef int32_t I4 __attribute__((ext_vector_type(4), aligned(4)));
    const int64_t per = (a.n + 3) / 4, at = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x;
    if (at >= a.m * per) return;
    const int64_t m = at / per, n = at % per * 4, width = GATED ? 2 * a.n : a.n;
    int32_t sum[2][4] = {};
    auto add = [&](const int32_t *p, int32_t (&s)[4]) {
        if (n + 4 <= a.n) {
            const I4 v = *(const I4 *)p;
#pragma unroll
            for (int e = 0; e < 4; e++) s[e] += v[e];
        } else {
#pragma unroll
            for (int e = 0; e < 3; e++)
                if (n + e < a.n) s[e] += p[e];
        }
    };
#pragma unroll 4
    for (int i = 0; i < slices; i++) {
        const int32_t *const p = part + ((int64_t)i * a.m + m) * width + n;
        add(p, sum[0]);
        if constexpr (GATED) add(p + a.n, sum[1]);
    }
    const float xs = a.xs[m];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (n + e >= a.n) continue;
        float y = scaled(sum[0][e], xs, a.ws[n + e], a.bias ? a.bias[n + e] : 0.f);
        if constexpr (GATED)
            y = gated(y, scaled(sum[1][e], xs, a.ws[a.n + n + e], a.bias ? a.bias[a.n + n + e] : 0.f), a.act);
        else if (a.act == ST_ACT_RELU)
            y = y < 0.f ? 0.f : y;
        ((T *)a.out)[m * a.out_stride + n + e] = (T)y;
    }
}

typedef Shape<256, 256, 128, 2> Large;
typedef Shape<128, 128, 64, 3> Middle;
typedef Shape<64, 128, 64, 4> Low;
typedef Shape<64, 64, 128, 3> Small;
typedef Shape<64, 64, 256, 4, true> Deep;
typedef Shape<64, 128, 128, 5, true> DeepLow;

enum Kernel { ONE, FEW, LARGE, MIDDLE, LOW, SMALL, DEEP, DEEP_LOW, ANY };

template <class F>
st_status with_shape(int kernel, F &&f) {
    switch (kernel) {
        case LARGE: return f(Large());
        case MIDDLE: return f(Middle());
        case LOW: return f(Low());
        case SMALL: return f(Small());
        case DEEP: return f(Deep());
        default: return f(DeepLow());
    }
}

struct Plan {
    int kernel, slices;
};

// Which kernel: the one whose time, in us, comes out least.  A workgroup takes `start`, and `unit` for each unit beside its stages, of
// which one takes `alone`, or `shared` where two workgroups of a CU run at once; or its bytes come at `rate` (MB a us) and take longer; slices cost
// their join, `join` and `each` of them, and the memory of their sums.  Fitted to the times of all kernels at 400 shapes, at 17 to 96 % of which a
// given one is not the fastest (256 x 256 tiles at the 244 of more than 64 rows, in stages of 128 k as they are); the choice costs
// 1.0 % over the fastest on average (0.6 % above 64 rows; most: 384 x 4096 x 11003, 45 us instead of 35, a tile and a half a CU).
struct Rates {
    int kernel, bm, bn, bk, shared_by;
    double start, unit, alone, shared, rate, join, each;
};
constexpr Rates RATES[] = {
    {LARGE, 256, 256, 128, 1, 3.49, 13.8, 1.351, 1.351, 2.28, 0, 0}, {MIDDLE, 128, 128, 64, 2, 4.37, 2.98, 0.307, 0.664, 3.62, 0, 0},
    {LOW, 64, 128, 64, 2, 3.13, 2.75, 0.264, 0.494, 8.4, 0, 0},    {SMALL, 64, 64, 128, 2, 3.95, 1.78, 0.307, 0.455, 3.44, 2.21, 0.446},
    {DEEP, 64, 64, 256, 1, 5.23, 1.48, 0.51, 0.51, 5.58, 2.22, 0.263}, {DEEP_LOW, 64, 128, 128, 1, 3.13, 3.58, 0.427, 0.427, 4.41, 0, 0},
};

// A tile's offsets are 32 bits: rows of weights up to 256 on, and in a gated product n further.
bool is_near(int64_t n, bool is_gated, int64_t x_stride, int64_t w_stride, int64_t out_stride) {
    return x_stride < 1 << 23 && out_stride < 1 << 21 && w_stride < 1 << 24 && ((is_gated ? n : 0) + 256) * w_stride < ((int64_t)1 << 32) - (1 << 16);
}

// tiles_too: offsets are near enough for the kernels with tiles.
Plan plan_of(int64_t m, int64_t k, int64_t n, bool is_gated, bool tiles_too) {
    const int64_t width = is_gated ? 2 * n : n, cus = st::device_cus();
    if (m <= 4 && k >= 512 && (m == 1 ? 1 : m == 2 ? 2 : 4) * k <= 64 * 1024) return Plan{ONE, 1};
    Plan best = {ANY, 1};
    double least = 1e300;
    for (const Rates &r : RATES) {
        if (!tiles_too) break;
        const bool once = r.kernel == DEEP || r.kernel == DEEP_LOW, narrow = r.kernel == SMALL || r.kernel == DEEP, halves = r.kernel == LOW || r.kernel == DEEP_LOW;
        if (once != (m <= 64) || (halves && !is_gated)) continue;
        const int64_t stages = (k + r.bk - 1) / r.bk, tiles = (m + r.bm - 1) / r.bm * ((width + r.bn - 1) / r.bn);
        for (const int slices : {1, 2, 3, 4, 6, 8, 12, 16}) {
            if (slices > 1 && (!narrow || slices > stages / 2 || tiles * slices > 5 * cus)) break;
            if (slices == 1 && narrow && is_gated) continue;
            const int64_t per = (tiles * slices + cus - 1) / cus, full = per / r.shared_by, rest = per % r.shared_by, of = (stages + slices - 1) / slices;
            double t = r.start + (double)full * (r.unit + (double)of * r.shared) + (rest ? r.unit + (double)of * r.alone : 0);
            t = std::max(t, r.start + ((double)m + (double)width) * (double)k / (1e6 * r.rate));
            if (slices > 1) t += r.join + r.each * slices + (double)m * (double)width * 4 * (slices + 1) / 4e6;
            if (t < least) least = t, best = Plan{r.kernel, slices};
        }
    }
    if (m <= 32 && width <= 1 << 26) {  // (a launch has less than 2^32 threads along x)
        const double blocks = (double)((width + 15) / 16), at_once = 8.0 * (double)cus / (is_gated ? 2 : 1);
        const double t = 4.61 + 0.134e-6 * (double)width * (double)k * (1 + 0.613 * (double)m / 16) + 0.69 * std::ceil(blocks / at_once) * (double)k / 1024;
        if (t < least) best = Plan{FEW, 1};
    }
    return best;
}

// The plan of rows of codes as short as 16-byte alignment leaves them and of a contiguous out: no others are nearer.
Plan plan_of(int64_t m, int64_t k, int64_t n, bool is_gated) {
    const int64_t stride = (k + 15) & ~(int64_t)15;
    return plan_of(m, k, n, is_gated, is_near(n, is_gated, stride, stride, n));
}

st_status product8(const char *name, const Product &a, int32_t dtype, bool is_gated, void *work, int64_t work_bytes, st_stream stream) {
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
    const Plan plan = vec ? plan_of(a.m, a.k, a.n, is_gated, is_near(a.n, is_gated, a.x_stride, a.w_stride, a.out_stride)) : Plan{ANY, 1};
    return st::with_dtype(dtype, [&](auto *t) -> st_status {
        using T = std::remove_pointer_t<decltype(t)>;
        typedef std::integral_constant<int, 1> I1;
        typedef std::integral_constant<int, 2> I2;
        typedef std::integral_constant<int, 4> I4;
        typedef std::integral_constant<int, 8> I8;
        if (plan.kernel == ONE) {
            const int rows = a.m == 1 ? 1 : a.m == 2 ? 2 : 4, lds = rows * (int)((a.k + 1023) / 1024 * 1024);
            auto go = [&](auto m_, auto r_, auto u_) {
                constexpr int M = decltype(m_)::value, R = decltype(r_)::value, U = decltype(u_)::value;
                const int64_t most = (int64_t)st::device_cus() * (M == 1 ? 64 : std::min(8, 160 * 1024 / lds));
                const uint32_t groups = (uint32_t)std::min<int64_t>((a.n + 4 * R - 1) / (4 * R), most);
                if (is_gated)
                    k_one8<T, true, M, R, U><<<groups, 256, lds, st::stream_of(stream)>>>(a);
                else
                    k_one8<T, false, M, R, U><<<groups, 256, lds, st::stream_of(stream)>>>(a);
            };
            // Rows of weights at once: two, for x's share of the LDS reads; one where there are few rows for all waves, and of long rows for
            // one row of x (us with one and two: 32768 x 8192 40.2 and 42, 1024 x 16384 7.2 and 8; 11003 x 4096 10.9 and 10.6).
            auto rows_of = [&](auto m_) {
                if (a.n <= 2048 || (a.m == 1 && a.k >= 8192))
                    go(m_, I1(), I8());
                else
                    go(m_, I2(), I4());
            };
            if (rows == 1)
                rows_of(I1());
            else if (rows == 2)
                rows_of(I2());
            else
                rows_of(I4());
            ST_LAUNCH_CHECK();
            return ST_OK;
        }
        if (plan.kernel == FEW) {
            auto go = [&](auto kernel, int mb, int waves) {
                kernel<<<dim3((uint32_t)((a.n + 15) / 16), (uint32_t)((a.m + 16 * mb - 1) / (16 * mb))), 64 * waves, 0, st::stream_of(stream)>>>(a);
            };
            if (a.m <= 16 && is_gated)
                go(k_few8<T, true, 1, 2, 4, 1>, 1, 4);
            else if (a.m <= 16)
                go(k_few8<T, false, 1, 1, 8, 4>, 1, 8);
            else if (is_gated)
                go(k_few8<T, true, 2, 2, 4, 1>, 2, 4);
            else
                go(k_few8<T, false, 2, 1, 8, 2>, 2, 8);
            ST_LAUNCH_CHECK();
            return ST_OK;
        }
        if (plan.kernel != ANY) {
            const int64_t width = is_gated ? 2 * a.n : a.n, need = plan.slices > 1 ? 4 * plan.slices * a.m * width : 0;
            if (need && (!work || work_bytes < need))
                return st::fail(ST_ERR_INVALID, "%s: %lld bytes of work memory are needed, got %lld", name, (long long)need, (long long)(work ? work_bytes : 0));
            const st_status status = with_shape(plan.kernel, [&](auto shape) -> st_status {
                using Tiles = decltype(shape);
                constexpr bool SLICED = std::is_same_v<Tiles, Small> || std::is_same_v<Tiles, Deep>, NARROW = SLICED;  // (a wave's columns are 32)
                constexpr bool HALVES = std::is_same_v<Tiles, Low> || std::is_same_v<Tiles, DeepLow>;
                auto go = [&](auto kernel, const Product &p, int bn) {
                    Units u;
                    const int64_t stages = (p.k + Tiles::BK - 1) / Tiles::BK;
                    u.slice = (int32_t)((stages + plan.slices - 1) / plan.slices), u.slices = (uint32_t)((stages + u.slice - 1) / u.slice);
                    u.tiles_m = (uint32_t)((p.m + Tiles::BM - 1) / Tiles::BM), u.tiles_n = (uint32_t)((p.n + bn - 1) / bn);
                    u.total = u.tiles_m * u.tiles_n * u.slices;
                    const uint32_t most = (uint32_t)(st::device_cus() * std::min(Tiles::AT_ONCE, 4));
                    kernel<<<std::min(u.total, most), 256, Tiles::LDS, st::stream_of(stream)>>>(p, u);
                    return (int32_t)u.slices;
                };
                if (plan.slices > 1) {
                    if constexpr (SLICED) {
                        Product p = a;
                        p.n = width, p.out = work;
                        const int32_t slices = go(k_product8<int32_t, false, Tiles>, p, Tiles::BN);
                        ST_LAUNCH_CHECK();
                        const int64_t blocks = (a.m * ((a.n + 3) / 4) + 255) / 256, along = std::min<int64_t>(blocks, 1 << 23);
                        const dim3 grid((uint32_t)along, (uint32_t)((blocks + along - 1) / along));
                        if (is_gated)
                            k_join8<T, true><<<grid, 256, 0, st::stream_of(stream)>>>(a, (const int32_t *)work, slices);
                        else
                            k_join8<T, false><<<grid, 256, 0, st::stream_of(stream)>>>(a, (const int32_t *)work, slices);
                    }
                } else if (is_gated) {
                    if constexpr (!NARROW) go(k_product8<T, true, Tiles>, a, Tiles::BN / 2);
                } else {
                    if constexpr (!HALVES) go(k_product8<T, false, Tiles>, a, Tiles::BN);
                }
                ST_LAUNCH_CHECK();
                return ST_OK;
            });
            return status;
        }
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

extern "C" int64_t st_matmul_8bit_bytes(int64_t m, int64_t k, int64_t n, int32_t is_gated) {
    if (m <= 0 || k <= 0 || n <= 0 || m > (int64_t)1 << 30 || k > 131072 || n > (int64_t)1 << 30) return 0;
    const Plan plan = plan_of(m, k, n, is_gated != 0);
    return plan.slices > 1 ? 4 * plan.slices * m * (is_gated ? 2 * n : n) : 0;
}

extern "C" st_status st_matmul_8bit_plan(int64_t m, int64_t k, int64_t n, int32_t is_gated, int64_t *plan) {
    st::clear_error();
    if (m <= 0 || k <= 0 || n <= 0 || m > (int64_t)1 << 30 || k > 131072 || n > (int64_t)1 << 30 || !plan)
        return st::fail(ST_ERR_INVALID, "matmul_8bit_plan: m %lld and n %lld (1 to 2^30), k %lld (1 to 131072)", (long long)m, (long long)n, (long long)k);
    const Plan p = plan_of(m, k, n, is_gated != 0);
    plan[0] = p.kernel, plan[1] = p.slices;
    return ST_OK;
}

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
