// 4-bit weights: the quantiser (the format is in quant4.h) and the products of a few rows with them.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "lanes.h"
#include "quant4.h"

namespace {

// One thread per 8 values; a group is 4, 8 or 16 neighbouring lanes.  `width`: 8-value units of a row (of all rows, where they
// lie behind each other).  Bound by HBM: 16384 x 8192 bf16 with values, 612 MB, 122 us (5.0 TB/s, a large copy's rate; 154 us
// with a 64-bit quotient for each value).
template <class T, int GROUP>
__global__ __launch_bounds__(256) void k_quantise4(const T *__restrict__ x, int64_t total, int64_t width, int64_t stride,
                                                   bool vec, uint32_t *__restrict__ codes, float2 *__restrict__ scales,
                                                   T *__restrict__ values, bool vec_values) {
    const int64_t first = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256, i = first + threadIdx.x;
    const bool used = i < total;
    float v[8] = {};
    if (used) {
        // The workgroup's first row is the same for all lanes (a scalar division); a lane's is a few rows on.
        int64_t row = first / width, at = first - row * width + threadIdx.x;
        if (width >= 256) {
            if (at >= width) at -= width, row++;
        } else {
            const uint32_t more = (uint32_t)at / (uint32_t)width;
            row += more, at -= more * width;
        }
        st::load8(x + row * stride + at * 8, vec, v);
    }
    float scale, lo;
    const uint32_t c = st::quantise8<GROUP / 8>(v, used, scale, lo);
    if (!used) return;
    codes[i] = c;
    if (threadIdx.x % (GROUP / 8) == 0) scales[i / (GROUP / 8)] = make_float2(scale, lo);
    if (values) {
        st::values8(c, scale, lo, v);
        st::store8(values + i * 8, vec_values, v);
    }
}

// Products of 16 MB rows of x with 16 NT rows of weights a workgroup, the sums over k shared by its four waves.
//
// y = sum over groups of s (sum x c) + lo (sum x).  The first sum runs on the matrix cores (16x16x32, f32 sums): x is one
// operand as it lies in memory (f16 and bf16), and a code is the f16 or bf16 number 16 + c, its four bits put under the
// exponent of 16 by a shift and a v_and_or (a VALU operation per code), so that sum x c = sum x (16 + c) - 16 sum x loses two
// bits of the f32 sum and not seven, as 1024 + c or 128 + c would.  sum x is one more product, with ones, which comes out
// in the lanes that want it.  f32 rows are three bf16 parts of 8 bits each, taken off one after the other without rounding, and
// codes beside them are taken less 8.
//
// Lane (i, q) of a wave reads 16 bytes (32 codes) of weight row i: 64 bytes of each of 16 rows a load.  For groups of 32
// and 64 a product over 32 k has to stay inside a group: the four lanes of a row exchange words (a 4 x 4 transposition by
// v_permlane swaps), so that lane q has the q-th 8 codes of each 32.  Lines of 128 bytes of codes are read whole while they are
// there (16 waves' rows are four times the L1 cache): two steps at once.  A row's scales come 8 groups at once into LDS, which the
// lanes of the row then read (16 groups at once take 16 registers more at 64 rows of weights, and 19 are put away: 23.5 us where
// 8 take 18.3, 11003 x 4096 in groups of 32).
//
// 32768 x 8192 and one row of bf16: 35 us (4.3 TB/s; the weights' bytes alone would take 23), 11003 x 4096 and 16 rows of f16:
// 18 (5).  Both wait for the issue of instructions rather than for memory: two waves to a SIMD at most, by their registers.
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

constexpr int STEP = 128;  // k of a wave's step

template <class T>
constexpr int parts_of() { return sizeof(T) == 4 ? 3 : 1; }

// One step's loads of a wave.
template <class T, int NT, int MB>
struct Step {
    u4 codes[NT];
    u4 x[MB][4][sizeof(T) / 2];  // 8 elements for each of the four products
};

template <class T>
__device__ __forceinline__ f4 product(u4 a, u4 b, f4 c) {
    if constexpr (std::is_same_v<T, _Float16>)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

// The upper halves (bf16 parts) of two f32 words, the first below.
__device__ __forceinline__ uint32_t upper_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302); }

// 8 codes as the products' operand, in the order 0 4 1 5 2 6 3 7.  Beside f16 and bf16 rows: 16 + c, the exponent of 16 with c
// in the upper four bits of the mantissa.  Beside f32's parts: (c - 8) / 16 in bf16 (twice the operations), as an f32 sum has
// no bits to spare for an offset (groups of 128 of 4096: 2.2e-6 off with 16 + c).
template <class T>
struct Numbers {
    uint32_t mask, exponent, ones;
    __device__ __forceinline__ Numbers() {
        if constexpr (std::is_same_v<T, _Float16>) {
            asm("s_mov_b32 %0, 0x03C003C0" : "=s"(mask));
            asm("v_mov_b32 %0, 0x4C004C00" : "=v"(exponent));
            ones = 0x3C003C00;
        } else {
            asm("s_mov_b32 %0, 0x00780078" : "=s"(mask));
            asm("v_mov_b32 %0, 0x41804180" : "=v"(exponent));
            ones = 0x3F803F80;
        }
    }
    __device__ __forceinline__ u4 operator()(uint32_t c) const {
        if constexpr (std::is_same_v<T, float>) {
            const uint32_t low = c ^ 0x88888888u, high = low >> 16;  // c - 8 in two's complement
            auto pair = [](uint32_t a, uint32_t b) {
                return upper_halves(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_off_f32_i4((int)a)),
                                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_off_f32_i4((int)b)));
            };
            return u4{pair(low, high), pair(low >> 4, high >> 4), pair(low >> 8, high >> 8), pair(low >> 12, high >> 12)};
        } else if constexpr (std::is_same_v<T, _Float16>) {
            return u4{((c << 6) & mask) | exponent, ((c << 2) & mask) | exponent, ((c >> 2) & mask) | exponent, ((c >> 6) & mask) | exponent};
        } else {
            return u4{((c << 3) & mask) | exponent, ((c >> 1) & mask) | exponent, ((c >> 5) & mask) | exponent, ((c >> 9) & mask) | exponent};
        }
    }
    // A group's scale and lowest value for sums over these numbers.
    static __device__ __forceinline__ float2 scaled(float2 pair) {
        if constexpr (std::is_same_v<T, float>)
            return make_float2(16.f * pair.x, __builtin_fmaf(8.f, pair.x, pair.y));
        else
            return make_float2(pair.x, __builtin_fmaf(-16.f, pair.x, pair.y));
    }
};

// Elements 0 1 .. 7 to the order 0 4 1 5 2 6 3 7 that a word's codes come out in.
__device__ __forceinline__ u4 in_code_order(u4 x) {
    return u4{__builtin_amdgcn_perm(x[2], x[0], 0x05040100), __builtin_amdgcn_perm(x[2], x[0], 0x07060302),
              __builtin_amdgcn_perm(x[3], x[1], 0x05040100), __builtin_amdgcn_perm(x[3], x[1], 0x07060302)};
}

// 8 elements as the products take them: in the codes' order, f32 in three parts.
template <class T>
__device__ __forceinline__ void parts8(const u4 (&x)[sizeof(T) / 2], u4 (&part)[parts_of<T>()]) {
    if constexpr (sizeof(T) == 2) {
        part[0] = in_code_order(x[0]);
    } else {
        constexpr int order[8] = {0, 4, 1, 5, 2, 6, 3, 7};
        uint32_t r[8];
#pragma unroll
        for (int e = 0; e < 8; e++) r[e] = x[order[e] >> 2][order[e] & 3];
#pragma unroll
        for (int p = 0; p < 3; p++) {
            part[p] = u4{upper_halves(r[0], r[1]), upper_halves(r[2], r[3]), upper_halves(r[4], r[5]), upper_halves(r[6], r[7])};
            if (p < 2) {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    r[e] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, r[e]) - __builtin_bit_cast(float, r[e] & 0xFFFF0000u));
            }
        }
    }
}

// One output as the definition has it, sum x (scale c + lo), by a whole wave; `nan`: x holds a NaN.
template <class T, int GROUP>
__device__ __forceinline__ float sum_of_values(const T *x, const uint8_t *codes, const float2 *scales, int k, int lane, bool &nan) {
    float sum = 0.f;
    bool bad = false;
    for (int u = lane; u < k / 8; u += 64) {
        float v[8], w[8];
        st::load8(x + 8 * u, false, v);
        const float2 pair = scales[u / (GROUP / 8)];
        st::values8(((const uint32_t *)codes)[u], pair.x, pair.y, w);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            bad = bad || v[i] != v[i];
            sum = __builtin_fmaf(v[i], w[i], sum);
        }
    }
    nan = __any(bad);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += st::xor_lane(sum, o, lane);
    return sum;
}

template <class T, int GROUP, int NT, int MB>
__global__ __launch_bounds__(256, 2) void k_matvec4(const T *__restrict__ x, int32_t m, int32_t k, int64_t x_stride,
                                                    const uint8_t *__restrict__ codes, const float2 *__restrict__ scales, int64_t n,
                                                    const float *__restrict__ bias, bool relu, T *__restrict__ out,
                                                    int64_t out_stride) {
    constexpr int PARTS = parts_of<T>(), G = STEP / GROUP, BLOCK = 8, PER_BLOCK = BLOCK / G;  // groups of a step, groups and steps of a block
    __shared__ float sums[4][16 * MB][16 * NT + 4];
    __shared__ float2 block[4][NT][16][BLOCK + 1];  // a wave's rows: BLOCK groups of each
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, q = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16 * NT;
    const int m0 = blockIdx.y * 16 * MB;
    const int steps = k / STEP, first = steps * wave / 4, last = steps * (wave + 1) / 4;

    // Where this lane's weights, scales and rows of x begin (rows past the end repeat the last one and are not stored), the first
    // two from the workgroup's first row on, in 32 bits: 64 rows of 2^20.
    const uint8_t *const w0 = codes + n0 * (k / 2);
    const float2 *const sc0 = scales + n0 * (k / GROUP);
    uint32_t w[NT], sc[NT];
    const T *xr[MB];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const uint32_t row = (uint32_t)min((int64_t)(16 * t + col), n - 1 - n0);
        w[t] = row * (uint32_t)(k / 2);
        sc[t] = row * (uint32_t)(k / GROUP);
    }
#pragma unroll
    for (int b = 0; b < MB; b++) xr[b] = x + min(m0 + 16 * b + col, m - 1) * x_stride;

    // (Rows of x need the alignment of their elements only: a load of 16 bytes may begin at any of them.)
    typedef uint32_t X4 __attribute__((ext_vector_type(4), aligned(2)));
    auto load = [&](auto tail_, int step, Step<T, NT, MB> &s) {
        constexpr bool tail = decltype(tail_)::value;  // the step may reach past k (which is a multiple of 32)
        const int k0 = step * STEP + 32 * q;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            s.codes[t] = tail && k0 >= k ? u4{0, 0, 0, 0} : *(const u4 *)(w0 + (w[t] + (uint32_t)(k0 / 2)));
        }
#pragma unroll
        for (int b = 0; b < MB; b++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                // Product j's 8 elements of this lane: the j-th 8 of its 32 codes, or after the exchange the q-th of the j-th 32.
                const int at = step * STEP + (GROUP == STEP ? 32 * q + 8 * j : 32 * j + 8 * q);
#pragma unroll
                for (int h = 0; h < (int)sizeof(T) / 2; h++)
                    s.x[b][j][h] = tail && at >= k ? u4{0, 0, 0, 0} : u4(*(const X4 *)((const char *)(xr[b] + at) + 16 * h));
            }
    };

    const Numbers<T> numbers;

    f4 acc[NT][MB];
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int b = 0; b < MB; b++) acc[t][b] = f4{0.f, 0.f, 0.f, 0.f};

    // `group`: of the block in LDS, the step's first.
    auto compute = [&](const Step<T, NT, MB> &s, int group) {
        u4 c[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            c[t] = s.codes[t];
            if constexpr (GROUP < STEP) {
                const auto a = __builtin_amdgcn_permlane32_swap(c[t][0], c[t][2], false, false);
                const auto d = __builtin_amdgcn_permlane32_swap(c[t][1], c[t][3], false, false);
                const auto e = __builtin_amdgcn_permlane16_swap(a[0], d[0], false, false);
                const auto f = __builtin_amdgcn_permlane16_swap(a[1], d[1], false, false);
                c[t] = u4{(uint32_t)e[0], (uint32_t)e[1], (uint32_t)f[0], (uint32_t)f[1]};
            }
        }
#pragma unroll
        for (int i = 0; i < G; i++) {
            f4 dot[NT][MB], sum[MB];
#pragma unroll
            for (int b = 0; b < MB; b++) {
                sum[b] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int t = 0; t < NT; t++) dot[t][b] = f4{0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (int j = i * (4 / G); j < (i + 1) * (4 / G); j++) {
                u4 xs[MB][PARTS];
#pragma unroll
                for (int b = 0; b < MB; b++) {
                    parts8<T>(s.x[b][j], xs[b]);
                }
#pragma unroll
                for (int p = 0; p < PARTS; p++)
#pragma unroll
                    for (int b = 0; b < MB; b++) sum[b] = product<T>(xs[b][p], u4{numbers.ones, numbers.ones, numbers.ones, numbers.ones}, sum[b]);
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const u4 y = numbers(c[t][j]);
#pragma unroll
                    for (int p = 0; p < PARTS; p++)
#pragma unroll
                        for (int b = 0; b < MB; b++) dot[t][b] = product<T>(xs[b][p], y, dot[t][b]);
                }
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const float2 pair = numbers.scaled(block[wave][t][col][group + i]);
                const float scale = pair.x, lo = pair.y;
#pragma unroll
                for (int b = 0; b < MB; b++)
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[t][b][r] = __builtin_fmaf(scale, dot[t][b][r], __builtin_fmaf(lo, sum[b][r], acc[t][b][r]));
            }
        }
    };

    // BLOCK groups from `from` on (those past the row's end repeat its last): lane (i, q) has the q-th fourth of row i's.
    float2 coming[NT][BLOCK / 4];
    const int groups = k / GROUP;
    auto load_block = [&](int from) {
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < BLOCK / 4; i++) coming[t][i] = sc0[sc[t] + (uint32_t)min(from + BLOCK / 4 * q + i, groups - 1)];
    };
    auto put_block = [&] {  // (a wave's LDS operations are carried out in order: no barrier)
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < BLOCK / 4; i++) block[wave][t][col][BLOCK / 4 * q + i] = coming[t][i];
    };
    // The next two steps' loads are under way while two are worked on (the last one's again behind the end: a condition around
    // them would make every wait one for all of them).
    if (first < last) {
        Step<T, NT, MB> s[2][2];
        load_block(first * G);
        load(std::false_type(), first, s[0][0]);
        load(std::false_type(), min(first + 1, last - 1), s[0][1]);
        for (int i = first; i < last; i += 4) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int at = i + 2 * j, group = (at - first) % PER_BLOCK * G;
                if (at >= last) break;
                if (group == 0) {
                    put_block();
                    load_block((at + PER_BLOCK) * G);
                }
                load(std::false_type(), min(at + 2, last - 1), s[1 - j][0]);
                load(std::false_type(), min(at + 3, last - 1), s[1 - j][1]);
                compute(s[j][0], group);
                if (at + 1 < last) compute(s[j][1], group + G);
            }
        }
    }
    if (wave == 3 && k % STEP) {  // (the groups of a part of a step are those of k's last)
        Step<T, NT, MB> s;
        load_block(k / STEP * G);
        load(std::true_type(), k / STEP, s);
        put_block();
        compute(s, 0);
    }

#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int b = 0; b < MB; b++)
#pragma unroll
            for (int r = 0; r < 4; r++) sums[wave][16 * b + 4 * q + r][16 * t + col] = acc[t][b][r];
    __syncthreads();
    for (int i0 = 64 * wave; i0 < 16 * MB * 16 * NT; i0 += 256) {
        const int i = i0 + lane, b = i / (16 * NT), j = i % (16 * NT);
        const bool used = m0 + b < m && n0 + j < n;
        float y = (sums[0][b][j] + sums[1][b][j]) + (sums[2][b][j] + sums[3][b][j]);
        // An infinity in x makes the two sums above infinities that cancel, and rows near the type's largest value pass f32's range
        // in them where their products with the weights do not: what is not finite is taken again from the definition (a row with
        // a NaN is NaN as it is).  11003 x 4096 and 16 rows of f16, 18 us: with one infinite row 210, with 16 of them 860.
        uint64_t odd = __ballot(used && !__builtin_isfinite(y));
        while (odd) {
            const int l = __ffsll((unsigned long long)odd) - 1, row = (i0 + l) / (16 * NT);
            const int64_t column = n0 + (i0 + l) % (16 * NT);
            bool nan;
            const float again = sum_of_values<T, GROUP>(x + (m0 + row) * x_stride, codes + column * (k / 2), scales + column * (k / GROUP), k, lane, nan);
            if (lane == l && !nan) y = again;
            odd &= nan ? __ballot(b != row) : ~(1ull << l);
        }
        if (!used) continue;
        if (bias) y += bias[n0 + j];
        if (relu && y < 0.f) y = 0.f;
        out[(m0 + b) * out_stride + n0 + j] = (T)y;
    }
}

}  // namespace

extern "C" st_status st_quantize_4bit(const void *x, int32_t dtype, int64_t n, int64_t k, int64_t x_stride,
                                      int64_t group, uint8_t *codes, float *scales, void *values, st_stream stream) {
    st::clear_error();
    if (n < 0 || k <= 0) return st::fail(ST_ERR_INVALID, "quantize_4bit: n %lld, k %lld", (long long)n, (long long)k);
    if (group != 32 && group != 64 && group != 128)
        return st::fail(ST_ERR_INVALID, "quantize_4bit: group %lld is none of 32, 64, 128", (long long)group);
    if (k % group)
        return st::fail(ST_ERR_INVALID, "quantize_4bit: k %lld is not a multiple of the group %lld",
                        (long long)k, (long long)group);
    if (x_stride < k)
        return st::fail(ST_ERR_INVALID, "quantize_4bit: rows of %lld elements lie %lld apart",
                        (long long)k, (long long)x_stride);
    if (n > (((int64_t)1 << 31) - 1) * 256 / (k / 8))
        return st::fail(ST_ERR_INVALID, "quantize_4bit: %lld x %lld values are too many for one call",
                        (long long)n, (long long)k);
    if (dtype < ST_F32 || dtype > ST_BF16)
        return st::fail(ST_ERR_INVALID, "quantize_4bit: dtype %d is none of ST_F32, ST_F16, ST_BF16",
                        (int)dtype);
    if (n == 0) return ST_OK;
    if (!x || !codes || !scales) return st::fail(ST_ERR_INVALID, "quantize_4bit: NULL buffer");
    const int64_t size = st::dtype_size(dtype);
    if (((uintptr_t)x | (uintptr_t)values) & (size - 1)) return st::fail(ST_ERR_INVALID, "quantize_4bit: x or values not aligned to its elements");
    if (((uintptr_t)codes & 3) || ((uintptr_t)scales & 7)) return st::fail(ST_ERR_INVALID, "quantize_4bit: codes are 4-byte, scales 8-byte aligned");
    if (!st::device_ok()) return ST_ERR_NO_DEVICE;
    const bool vec = st::rows_aligned(x, x_stride, size), vec_values = ((uintptr_t)values & 15) == 0;
    const int64_t total = n * (k / 8), blocks = (total + 255) / 256, along = std::min<int64_t>(blocks, 1 << 23);  // (below 2^32 threads)
    const dim3 grid((uint32_t)along, (uint32_t)((blocks + along - 1) / along));
    const int64_t width = x_stride == k ? total : k / 8;
    return st::with_dtype(dtype, [&](auto *t) -> st_status {
        using T = std::remove_pointer_t<decltype(t)>;
        auto go = [&](auto kernel) {
            kernel<<<grid, 256, 0, st::stream_of(stream)>>>((const T *)x, total, width, x_stride, vec, (uint32_t *)codes,
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
    if (m < 0 || k <= 0 || n < 0)
        return st::fail(ST_ERR_INVALID, "matvec_4bit: m %lld, k %lld, n %lld",
                        (long long)m, (long long)k, (long long)n);
    if (group != 32 && group != 64 && group != 128)
        return st::fail(ST_ERR_INVALID, "matvec_4bit: group %lld is none of 32, 64, 128", (long long)group);
    if (k % group)
        return st::fail(ST_ERR_INVALID, "matvec_4bit: k %lld is not a multiple of the group %lld",
                        (long long)k, (long long)group);
    if (m > 1 << 19 || k > 1 << 20 || n > 1 << 28)  // (a launch holds less than 2^32 threads along x, 2^16 workgroups along y)
        return st::fail(ST_ERR_INVALID, "matvec_4bit: m %lld (up to 2^19), k %lld (up to 2^20), n %lld (up to 2^28)",
                        (long long)m, (long long)k, (long long)n);
    if (x_stride < k || out_stride < n)
        return st::fail(ST_ERR_INVALID, "matvec_4bit: rows of %lld and %lld elements lie %lld and %lld apart",
                        (long long)k, (long long)n, (long long)x_stride, (long long)out_stride);
    if (dtype < ST_F32 || dtype > ST_BF16)
        return st::fail(ST_ERR_INVALID, "matvec_4bit: dtype %d is none of ST_F32, ST_F16, ST_BF16",
                        (int)dtype);
    if (m == 0 || n == 0) return ST_OK;
    if (!x || !codes || !scales || !out) return st::fail(ST_ERR_INVALID, "matvec_4bit: NULL buffer");
    const int64_t size = st::dtype_size(dtype);
    if (((uintptr_t)x | (uintptr_t)out) & (size - 1)) return st::fail(ST_ERR_INVALID, "matvec_4bit: x or out not aligned to its elements");
    if (((uintptr_t)codes & 15) || ((uintptr_t)scales & 7) || ((uintptr_t)bias & 3))
        return st::fail(ST_ERR_INVALID, "matvec_4bit: codes are 16-byte, scales 8-byte, bias 4-byte aligned");
    if (!st::device_ok()) return ST_ERR_NO_DEVICE;
    return st::with_dtype(dtype, [&](auto *t) -> st_status {
        using T = std::remove_pointer_t<decltype(t)>;
        auto go = [&](auto kernel, int nt, int mb) {
            const dim3 grid((uint32_t)((n + 16 * nt - 1) / (16 * nt)), (uint32_t)((m + 16 * mb - 1) / (16 * mb)));
            kernel<<<grid, 256, 0, st::stream_of(stream)>>>((const T *)x, (int32_t)m, (int32_t)k, x_stride, codes, (const float2 *)scales, n,
                                                            bias, relu != 0, (T *)out, out_stride);
        };
        auto pick = [&](auto group_) {
            constexpr int GROUP = decltype(group_)::value;
            // Rows of weights a workgroup (16 NT): with more of them x is read and summed less often, with fewer a workgroup takes
            // less time.  So the fewest that leave the chip one workgroup a CU at most; where none does, 64 (for two blocks of
            // x 32, with both in one workgroup; f32's three parts leave registers for 32, and 16 rows of x at a time).  us at NT 1,
            // 2, 4, then 2 with two blocks, k = 4096 in groups of 128, bf16:
            //   n =        2048                3000 to 4096         6000 to 8192         11003                16384
            //   1 row      6.0 7.4 10.8        6.4 7.5 11.0         9.1 7.9 11.2         12.0 12.2 11.4       14.9 12.4 11.8
            //   16 rows    9.2 10.8 14.2       9.6 10.9 14.3        15.8 11.1 14.5       22.0 18.7 14.7       27.7 18.9 15.2
            //   32 rows    9.5 10.9 14.3 15.5  15.8 11.1 14.4 15.7  27.4 18.6 14.8 15.8  38.9 26.0 25.4 27.4  50.0 33.0 26.2 27.3
            // (17 rows at 11003: 29.2 22.7 22.4 20.9.)  f32, groups of 64, 16 rows: 14.5 and 18.6 at 4096, 25.3 and 18.8 at 6000.
            // Groups of 32 and k = 512 turn at the same n, but for one row of f16 in groups of 32 from 11003 on (14.0 16.1 17.0).
            const int64_t cus = st::device_cus(), tall = (m + 15) / 16;
            if ((n + 15) / 16 * tall <= cus) return go(k_matvec4<T, GROUP, 1, 1>, 1, 1);
            if (sizeof(T) == 4 || (n + 31) / 32 * tall <= cus) return go(k_matvec4<T, GROUP, 2, 1>, 2, 1);
            if constexpr (sizeof(T) == 2) {
                if (m > 16)
                    go(k_matvec4<T, GROUP, 2, 2>, 2, 2);
                else
                    go(k_matvec4<T, GROUP, 4, 1>, 4, 1);
            }
        };
        if (group == 32)
            pick(std::integral_constant<int, 32>());
        else if (group == 64)
            pick(std::integral_constant<int, 64>());
        else
            pick(std::integral_constant<int, 128>());
        ST_LAUNCH_CHECK();
        return ST_OK;
    });
}
