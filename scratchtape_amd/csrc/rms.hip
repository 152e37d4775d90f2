// The root-mean-square norm with the residual's addition, its 8-bit form, its backward pass, and the 8-bit row quantiser.
//
//   h = T(x + residual);  rstd = 1 / sqrt(mean h^2 + eps);  y = T(h rstd w)
//   8-bit rows: t = h w, a = max |t|, scale = f32(a rstd / 127), code = round_half_even(127 t / a)
//
// rstd is a factor of every value of a row, so it cancels in the codes: they depend on neither eps nor the order in which the
// squares are summed, and one pass over the row in registers finds both the sum and the maximum.  The quantiser is the same
// kernel with t = x and rstd = 1.
//
// Squares and products t are taken in 64 bits (exact for f32 values: squares of 1e30 do not overflow, and t decides codes); outputs
// are rounded to f32 and from there to their type (16-bit ones are off by half a step and 2^-24).  A row lies in the registers of TPR
// threads, V vectors of eight elements each; wider rows (V = 0) are read twice.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.h"
#include "lanes.h"
#include "quant8.h"

namespace {

constexpr int threads_of(int tpr) { return tpr == 64 ? 256 : tpr; }

__device__ __forceinline__ double wave_sum(double v) {
    const int lane = st::lane_id();
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += st::xor_lane(v, o, lane);
    return v;
}

__device__ __forceinline__ double wave_max(double v) {
    const int lane = st::lane_id();
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmax(v, st::xor_lane(v, o, lane));
    return v;
}

struct Norm {
    const void *x, *residual, *w;
    int64_t rows, d, x_stride, r_stride;
    double eps;
    void *h;
    float *rstd;
    void *y;
    int8_t *codes;
    int64_t c_stride, c_width;  // c_width: bytes of a row of codes that are written, zeros behind d among them
    float *scales;
    void *values;
};

// Bound by HBM for many rows: 8191 x 8192 bf16 with residual to h, codes and values 118 to 130 us, 4.6 to 5.1 TB/s (a copy 4.95); the
// quantiser with values of 16384 x 8192 bf16 118 to 131 us, 5.1 to 5.7.  For few by one load's latency, the sum over the
// row's waves and a store's: 128 x 256 f32 3.5 us, 64 x 8192 bf16 7.
template <class T, class W, int TPR, int V, bool NORM>
__global__ __launch_bounds__(threads_of(TPR)) void k_rms(Norm a) {
    constexpr int ROWS = threads_of(TPR) / TPR, WAVES = TPR / 64, HELD = V ? V : 1;
    static_assert(ROWS == 1 || WAVES == 1, "rows of several waves meet at barriers");
    constexpr bool WIDE = V == 0;
    typedef st::Eight_t<T> T8;
    const int t = threadIdx.x % TPR, wave = t >> 6;
    const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * ROWS + threadIdx.x / TPR;
    if (row >= a.rows) return;  // (whole waves; with several waves a row the whole workgroup)
    const T *const x = (const T *)a.x + row * a.x_stride;
    const T *const r = NORM && a.residual ? (const T *)a.residual + row * a.r_stride : nullptr;
    const W *const w = (const W *)a.w;
    const int64_t span = (int64_t)TPR * 8 * HELD, passes = WIDE ? (a.d + span - 1) / span : 1;
    const bool eight = a.codes != nullptr;

    T8 h[HELD];
    auto fetch = [&](int64_t from) {
#pragma unroll
        for (int v = 0; v < HELD; v++) h[v] = st::load_eight(x, from + (v * TPR + t) * 8, a.d);
        if (r) {
            T8 e[HELD];
#pragma unroll
            for (int v = 0; v < HELD; v++) e[v] = st::load_eight(r, from + (v * TPR + t) * 8, a.d);
#pragma unroll
            for (int v = 0; v < HELD; v++)
#pragma unroll
                for (int i = 0; i < 8; i++) h[v][i] = (T)((float)h[v][i] + (float)e[v][i]);
        }
    };
    // t of vector v, in 64 bits.
    auto scaled = [&](int64_t at, T8 hv, double (&tv)[8]) {
        if constexpr (NORM) {
            const st::Eight_t<W> wv = st::load_eight(w, at, a.d);
#pragma unroll
            for (int i = 0; i < 8; i++) tv[i] = (double)(float)hv[i] * (double)(float)wv[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) tv[i] = (double)(float)hv[i];
        }
    };

    double sum = 0.0, top = 0.0;  // top: infinite where a value is not finite
    for (int64_t p = 0; p < passes; p++) {
        const int64_t from = p * span;
        fetch(from);
#pragma unroll
        for (int v = 0; v < HELD; v++) {
            const int64_t at = from + (v * TPR + t) * 8;
            if constexpr (NORM) {
                if (a.h && (at < a.d)) st::store_eight((T *)a.h + row * a.d, at, a.d, h[v]);
#pragma unroll
                for (int i = 0; i < 8; i++) sum = __builtin_fma((double)(float)h[v][i], (double)(float)h[v][i], sum);
            }
            if (eight) {
                double tv[8];
                scaled(at, h[v], tv);
#pragma unroll
                for (int i = 0; i < 8; i++) top = tv[i] - tv[i] == 0.0 ? fmax(top, __builtin_fabs(tv[i])) : INFINITY;
            }
        }
    }
    if constexpr (NORM) sum = wave_sum(sum);
    if (eight) top = wave_max(top);
    if constexpr (WAVES > 1) {
        __shared__ double sums[WAVES], tops[WAVES];
        if ((t & 63) == 0) sums[wave] = sum, tops[wave] = top;
        __syncthreads();
        sum = sums[0], top = tops[0];
#pragma unroll
        for (int i = 1; i < WAVES; i++) sum += sums[i], top = fmax(top, tops[i]);
    }
    const double rstd = NORM ? 1.0 / sqrt(sum / (double)a.d + a.eps) : 1.0;
    const bool finite = top < INFINITY;
    const float scale = finite ? (float)(top * rstd / 127.0) : NAN;
    if (t == 0) {
        if (NORM && a.rstd) a.rstd[row] = (float)rstd;
        if (eight) a.scales[row] = scale;
    }
    const st::RowCodes codes_of(finite ? top : 0.0);

    for (int64_t p = 0; p < passes; p++) {
        const int64_t from = p * span;
        if constexpr (WIDE) fetch(from);
#pragma unroll
        for (int v = 0; v < HELD; v++) {
            const int64_t at = from + (v * TPR + t) * 8;
            double tv[8];
            scaled(at, h[v], tv);
            T8 out;
            if (NORM && a.y) {
#pragma unroll
                for (int i = 0; i < 8; i++) out[i] = (T)(float)(tv[i] * rstd);
                st::store_eight((T *)a.y + row * a.d, at, a.d, out);
            }
            if (eight) {
                const uint2 c = finite ? codes_of(tv) : make_uint2(0, 0);  // (0 past the row's end)
                if (at + 8 <= a.c_width) {
                    typedef uint32_t C2 __attribute__((ext_vector_type(2), aligned(1)));
                    *(C2 *)(a.codes + row * a.c_stride + at) = C2{c.x, c.y};
                } else {
#pragma unroll
                    for (int i = 0; i < 7; i++)
                        if (at + i < a.c_width) a.codes[row * a.c_stride + at + i] = (int8_t)((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
                }
                if (a.values) {
#pragma unroll
                    for (int i = 0; i < 8; i++) out[i] = st::code_value<T>(c, i, scale);
                    st::store_eight((T *)a.values + row * a.d, at, a.d, out);
                }
            }
        }
    }
}

template <class T, class W, bool NORM>
st_status launch_rms(const Norm &a, hipStream_t stream) {
    auto go = [&](auto kernel, int tpr) -> st_status {
        const int64_t per = threads_of(tpr) / tpr, blocks = (a.rows + per - 1) / per, along = std::min<int64_t>(blocks, 1 << 21);
        const dim3 grid((uint32_t)along, (uint32_t)((blocks + along - 1) / along));
        kernel<<<grid, threads_of(tpr), 0, stream>>>(a);
        ST_LAUNCH_CHECK();
        return ST_OK;
    };
    // The width of a row of codes counts too: its zeros are written with it.  Threads of a row: as few as hold it, so that many rows are
    // on their way on a CU; for few rows more of them (us with 256 and 1024 threads: 8191 rows of 8192 bf16 to 8 bits 129 and 167, 64
    // of them 10.1 and 7.5; 2000 rows of 16384 f16 with 512 and 1024 67 and 77, 515 of 11003 14.6 and 14.2).
    const int64_t wide = std::max(a.d, a.c_width);
    const bool many = a.rows >= 2 * st::device_cus();
    if (wide <= 512) return go(k_rms<T, W, 64, 1, NORM>, 64);
    if (wide <= 1024) return go(k_rms<T, W, 64, 2, NORM>, 64);
    if (wide <= 2048) return go(k_rms<T, W, 128, 2, NORM>, 128);
    if (wide <= 4096) return go(k_rms<T, W, 256, 2, NORM>, 256);
    if (wide <= 8192 && many) return go(k_rms<T, W, 256, 4, NORM>, 256);
    if (wide <= 8192) return go(k_rms<T, W, 1024, 1, NORM>, 1024);
    if (wide <= 16384 && many) return go(k_rms<T, W, 512, 4, NORM>, 512);
    if (wide <= 16384) return go(k_rms<T, W, 1024, 2, NORM>, 1024);
    return go(k_rms<T, W, 1024, 0, NORM>, 1024);
}

struct Back {
    const void *dy, *h, *dh, *w;
    const float *rstd;
    int64_t rows, d, dy_stride, h_stride, dh_stride;
    void *dx;
    float *part;  // [gridDim.x, d]: the workgroups' sums of dy h rstd (the gradient itself where there is one workgroup)
};

// dx = dh + rstd (g - xh mean(g xh)) with g = dy w, xh = h rstd; a workgroup's rows are blockIdx.x ROWS .. in steps of
// gridDim.x ROWS, and a thread keeps the weight gradient's sums of its own columns over them in 64 bits, so that their error does not
// grow with the number of rows (chains of 64 rows in f32 are off by 1.5e-7, 4.4e-8 so; 32768 x 256 bf16 25 us, 24 with f32 sums); each
// part is rounded to f32 once.  Where those sums leave too few registers, or room for one workgroup of a CU's two, the weights lie in LDS (us
// so and in registers: 2000 x 16384 f32 114 and 131, 8000 x 1900 bf16 32 and 40; f32, which has one workgroup a CU, 64 and 61).
// Bound by HBM: 16384 x 4096 bf16 with dh 110 us with the sum's launch, 4.9 TB/s; 4096 x 256 f32 11.2, latencies of rows one after the other.
template <class T, class W, int TPR, int V>
__global__ __launch_bounds__(threads_of(TPR)) void k_rms_back(Back a) {
    constexpr int ROWS = threads_of(TPR) / TPR, WAVES = TPR / 64;
    static_assert(ROWS == 1 || WAVES == 1, "rows of several waves meet at barriers");
    typedef st::Eight_t<T> T8;
    constexpr bool W_LDS = (V == 4 && sizeof(T) == 2) || (TPR == 1024 && V == 2);
    typedef float F4 __attribute__((ext_vector_type(4)));
    __shared__ F4 w_lds[W_LDS ? 2 * V : 1][TPR];
    const int t = threadIdx.x % TPR, wave = t >> 6, mine = threadIdx.x / TPR;
    float w_held[W_LDS ? 1 : V][8];
    double dw[V][8];
#pragma unroll
    for (int v = 0; v < V; v++) {
        const st::Eight_t<W> wv = st::load_eight((const W *)a.w, (v * TPR + t) * 8, a.d);
#pragma unroll
        for (int i = 0; i < 8; i++) dw[v][i] = 0;
        if constexpr (W_LDS) {
            if (mine == 0) {
#pragma unroll
                for (int i = 0; i < 2; i++) w_lds[2 * v + i][t] = F4{(float)wv[4 * i], (float)wv[4 * i + 1], (float)wv[4 * i + 2], (float)wv[4 * i + 3]};
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) w_held[v][i] = (float)wv[i];
        }
    }
    if constexpr (W_LDS && ROWS > 1) __syncthreads();  // (else a thread reads what it wrote)
    auto weights = [&](int v, float (&w)[8]) {
        if constexpr (W_LDS) asm volatile("" ::: "memory");  // (from LDS each time, not into registers ahead of the loop)
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = W_LDS ? w_lds[2 * v + i / 4][t][i % 4] : w_held[W_LDS ? 0 : v][i];
    };
    // A row's last vector, of 16-bit elements, as its last eight, moved to their places when all loads are on their way (us so and with
    // load_eight: 8000 x 4003 bf16 64 and 99, 8000 x 1111 26 and 30, 16384 x 4096 109 and 109; f32 16384 x 4096, another day, 305 and 203).
    constexpr bool LATE = sizeof(T) == 2;
    auto load = [&](const T *row, int v) {
        const int64_t at = (v * TPR + t) * 8;
        return LATE ? st::load_raw(row, at, a.d) : st::load_eight(row, at, a.d);
    };
    auto settle = [&](T8 &x, int v) {
        if constexpr (LATE) st::settle<T>(x, (v * TPR + t) * 8, a.d);
    };
    __shared__ double sums[2][WAVES];
    int turn = 0;
    for (int64_t row = (int64_t)blockIdx.x * ROWS + mine; row < a.rows; row += (int64_t)gridDim.x * ROWS) {
        T8 dy[V], h[V], dh[V];
#pragma unroll
        for (int v = 0; v < V; v++) {
            dy[v] = load((const T *)a.dy + row * a.dy_stride, v);
            h[v] = load((const T *)a.h + row * a.h_stride, v);
            if (a.dh) dh[v] = load((const T *)a.dh + row * a.dh_stride, v);
        }
        const float rstd = a.rstd[row];
#pragma unroll
        for (int v = 0; v < V; v++) {
            settle(dy[v], v), settle(h[v], v);
            if (a.dh) settle(dh[v], v);
        }
        double s = 0.0;
#pragma unroll
        for (int v = 0; v < V; v++) {
            float w[8];
            weights(v, w);
#pragma unroll
            for (int i = 0; i < 8; i++) s = __builtin_fma((double)((float)dy[v][i] * w[i]), (double)(float)h[v][i], s);
        }
        s = wave_sum(s);
        if constexpr (WAVES > 1) {
            if ((t & 63) == 0) sums[turn][wave] = s;
            __syncthreads();
            s = sums[turn][0];
#pragma unroll
            for (int i = 1; i < WAVES; i++) s += sums[turn][i];
            turn ^= 1;  // (a wave is at most one row ahead of the others: two sets)
        }
        const float mean = (float)(s * (double)rstd / (double)a.d);
#pragma unroll
        for (int v = 0; v < V; v++) {
            T8 out;
            float w[8];
            weights(v, w);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float xh = (float)h[v][i] * rstd, g = (float)dy[v][i];
                dw[v][i] = __builtin_fma((double)g, (double)xh, dw[v][i]);
                const float dx = rstd * __builtin_fmaf(-xh, mean, g * w[i]);
                out[i] = (T)(a.dh ? (float)dh[v][i] + dx : dx);
            }
            st::store_eight((T *)a.dx + row * a.d, (v * TPR + t) * 8, a.d, out);
        }
    }
    if constexpr (ROWS > 1) {
        __shared__ double rows_of[ROWS - 1][V][8][TPR];
        if (mine > 0) {
#pragma unroll
            for (int v = 0; v < V; v++)
#pragma unroll
                for (int i = 0; i < 8; i++) rows_of[mine - 1][v][i][t] = dw[v][i];
        }
        __syncthreads();
        if (mine > 0) return;
#pragma unroll
        for (int m = 0; m < ROWS - 1; m++)
#pragma unroll
            for (int v = 0; v < V; v++)
#pragma unroll
                for (int i = 0; i < 8; i++) dw[v][i] += rows_of[m][v][i][t];
    }
#pragma unroll
    for (int v = 0; v < V; v++) {
        st::Eight_t<float> out;
#pragma unroll
        for (int i = 0; i < 8; i++) out[i] = (float)dw[v][i];
        st::store_eight(a.part + blockIdx.x * a.d, (v * TPR + t) * 8, a.d, out);
    }
}

// Rows too wide for a workgroup's registers: the gradient of the rows, one row a workgroup, read twice ..
template <class T, class W>
__global__ __launch_bounds__(1024) void k_rms_back_wide(Back a) {
    __shared__ double sums[16];
    const int64_t row = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (row >= a.rows) return;
    const T *const dy = (const T *)a.dy + row * a.dy_stride, *const h = (const T *)a.h + row * a.h_stride;
    const T *const dh = a.dh ? (const T *)a.dh + row * a.dh_stride : nullptr;
    const W *const w = (const W *)a.w;
    const float rstd = a.rstd[row];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < a.d; i += 1024) s = __builtin_fma((double)((float)dy[i] * (float)w[i]), (double)(float)h[i], s);
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.0;
    for (int i = 0; i < 16; i++) s += sums[i];
    const float mean = (float)(s * (double)rstd / (double)a.d);
    for (int64_t i = threadIdx.x; i < a.d; i += 1024) {
        const float dx = rstd * __builtin_fmaf(-(float)h[i] * rstd, mean, (float)dy[i] * (float)w[i]);
        ((T *)a.dx)[row * a.d + i] = (T)(dh ? (float)dh[i] + dx : dx);
    }
}

// .. and the sums of dy h rstd over the rows blockIdx.y, blockIdx.y + gridDim.y, .. of a column a thread.
template <class T>
__global__ __launch_bounds__(256) void k_rms_back_columns(Back a) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= a.d) return;
    double s = 0.0;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y)
        s = __builtin_fma((double)(float)((const T *)a.dy)[row * a.dy_stride + i], (double)((float)((const T *)a.h)[row * a.h_stride + i] * a.rstd[row]), s);
    a.part[blockIdx.y * a.d + i] = (float)s;
}

// dw[i] = sum over p of part[p, i]: 16 columns a workgroup, whose 64 rows of lanes take every 64th p, joined in order, in 64 bits.
// A launch's latency and one of the loads' (4096 x 256 f32's whole backward 3 us less than with 64 columns a workgroup).
__global__ __launch_bounds__(1024) void k_rms_back_sum(const float *__restrict__ part, int64_t parts, int64_t d, float *__restrict__ dw) {
    __shared__ double sums[16][16];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, column = lane & 15;
    const int64_t i = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 16 + column;
    double s = 0.0;
    if (i < d)
        for (int64_t p = threadIdx.x >> 4; p < parts; p += 64 * 8) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = p + 64 * j < parts ? part[(p + 64 * j) * d + i] : 0.f;
#pragma unroll
            for (int j = 0; j < 8; j++) s += (double)v[j];
        }
    s += st::xor_lane(s, 16, lane);
    s += st::xor_lane(s, 32, lane);
    if (lane < 16) sums[wave][column] = s;
    __syncthreads();
    if (threadIdx.x >= 16 || i >= d) return;
#pragma unroll
    for (int j = 1; j < 16; j++) s += sums[j][column];
    dw[i] = (float)s;
}

// Its grid: a launch has less than 2^32 threads along x.
dim3 sum_grid(int64_t d) {
    const int64_t blocks = (d + 15) / 16, along = std::min<int64_t>(blocks, 1 << 21);
    return dim3((uint32_t)along, (uint32_t)((blocks + along - 1) / along));
}

constexpr int64_t BACK_WIDEST = 16384;  // columns that a workgroup's registers hold

// Row lanes of a workgroup of k_rms_back, and the parts that its launch leaves to be summed: two workgroups a CU, one where its rows keep
// that busy (wide f32 rows, 1024 threads).  us with one and two: 4096 x 256 f32 12.2, 11.2, 8000 x 1900 61, 65, 16384 x 4096 188, 201;
// bf16 32768 x 512 44, 31, 8000 x 1111 33, 25, 16384 x 2048 66, 56, 16384 x 4096 131, 108, 4096 x 8192 60, 64.
int64_t back_rows(int64_t d) { return d <= 2048 ? 4 : 1; }
int64_t back_parts(int64_t rows, int64_t d, int64_t size) {
    if (d > BACK_WIDEST) return std::min<int64_t>((rows + 31) / 32, 64);
    const int64_t per = back_rows(d), groups = (rows + per - 1) / per;
    return std::min<int64_t>(groups, (d <= (size == 4 ? 1024 : 4096) ? 2 : 1) * st::device_cus());
}

template <class T, class W>
st_status launch_back(Back a, float *dw, hipStream_t stream) {
    const int64_t parts = back_parts(a.rows, a.d, sizeof(T));
    float *const part = a.part;
    if (parts == 1) a.part = dw;
    if (a.d > BACK_WIDEST) {
        const int64_t along = std::min<int64_t>(a.rows, 1 << 21);
        k_rms_back_wide<T, W><<<dim3((uint32_t)along, (uint32_t)((a.rows + along - 1) / along)), 1024, 0, stream>>>(a);
        ST_LAUNCH_CHECK();
        k_rms_back_columns<T><<<dim3((uint32_t)((a.d + 255) / 256), (uint32_t)parts), 256, 0, stream>>>(a);
    } else {
        auto go = [&](auto kernel, int tpr) { kernel<<<(uint32_t)parts, threads_of(tpr), 0, stream>>>(a); };
        if (a.d <= 512)
            go(k_rms_back<T, W, 64, 1>, 64);
        else if (a.d <= 1024)
            go(k_rms_back<T, W, 64, 2>, 64);
        else if (a.d <= 2048)
            go(k_rms_back<T, W, 64, 4>, 64);
        else if (a.d <= 4096)
            go(k_rms_back<T, W, 256, 2>, 256);
        else if (a.d <= 8192)
            go(k_rms_back<T, W, 1024, 1>, 1024);
        else
            go(k_rms_back<T, W, 1024, 2>, 1024);
    }
    ST_LAUNCH_CHECK();
    if (parts > 1) {
        k_rms_back_sum<<<sum_grid(a.d), 1024, 0, stream>>>(part, parts, a.d, dw);
        ST_LAUNCH_CHECK();
    }
    return ST_OK;
}

// f with null pointers of x's and the weight's element types: the weight's is x's or f32.
template <class F>
st_status with_types(int32_t dtype, int32_t w_dtype, F &&f) {
    return st::with_dtype(dtype, [&](auto *t) -> st_status {
        if (w_dtype == dtype) return f(t, t);
        return f(t, (float *)nullptr);
    });
}

bool unaligned(const void *p, int64_t size) { return ((uintptr_t)p & (size - 1)) != 0; }

constexpr int64_t MOST_ROWS = (int64_t)1 << 36, MOST_D = (int64_t)1 << 30;

}  // namespace

extern "C" st_status st_quantize_8bit(const void *x, int32_t dtype, int64_t n, int64_t k, int64_t x_stride, int8_t *codes,
                                      int64_t codes_stride, float *scales, void *values, st_stream stream) {
    st::clear_error();
    if (n < 0 || k <= 0 || n > MOST_ROWS || k > MOST_D)
        return st::fail(ST_ERR_INVALID, "quantize_8bit: n %lld (up to 2^36), k %lld (1 to 2^30)", (long long)n, (long long)k);
    if (x_stride < k || codes_stride < k)
        return st::fail(ST_ERR_INVALID, "quantize_8bit: rows of %lld elements lie %lld apart, their codes %lld", (long long)k,
                        (long long)x_stride, (long long)codes_stride);
    if (dtype < ST_F32 || dtype > ST_BF16) return st::fail(ST_ERR_INVALID, "quantize_8bit: dtype %d is none of ST_F32, ST_F16, ST_BF16", (int)dtype);
    if (n == 0) return ST_OK;
    if (!x || !codes || !scales) return st::fail(ST_ERR_INVALID, "quantize_8bit: NULL buffer");
    const int64_t size = st::dtype_size(dtype);
    if (unaligned(x, size) || unaligned(values, size) || unaligned(scales, 4))
        return st::fail(ST_ERR_INVALID, "quantize_8bit: x, values or scales not aligned to their elements");
    if (!st::device_ok()) return ST_ERR_NO_DEVICE;
    Norm a = {};
    a.x = x, a.rows = n, a.d = k, a.x_stride = x_stride;
    a.codes = codes, a.c_stride = codes_stride, a.c_width = std::min(codes_stride, (k + 15) & ~(int64_t)15);
    a.scales = scales, a.values = values;
    return st::with_dtype(dtype, [&](auto *t) -> st_status {
        using T = std::remove_pointer_t<decltype(t)>;
        return launch_rms<T, T, false>(a, st::stream_of(stream));
    });
}

extern "C" st_status st_rms_norm(const void *x, const void *residual, int32_t dtype, int64_t rows, int64_t d, int64_t x_stride,
                                 int64_t residual_stride, const void *weight, int32_t weight_dtype, float eps, void *h, float *rstd,
                                 void *y, int8_t *codes, int64_t codes_stride, float *scales, void *values, st_stream stream) {
    st::clear_error();
    if (rows < 0 || d <= 0 || rows > MOST_ROWS || d > MOST_D)
        return st::fail(ST_ERR_INVALID, "rms_norm: rows %lld (up to 2^36), d %lld (1 to 2^30)", (long long)rows, (long long)d);
    if (x_stride < d || (residual && residual_stride < d) || (codes && codes_stride < d))
        return st::fail(ST_ERR_INVALID, "rms_norm: rows of %lld elements lie %lld apart, the residual's %lld, their codes %lld", (long long)d,
                        (long long)x_stride, (long long)residual_stride, (long long)codes_stride);
    if (dtype < ST_F32 || dtype > ST_BF16) return st::fail(ST_ERR_INVALID, "rms_norm: dtype %d is none of ST_F32, ST_F16, ST_BF16", (int)dtype);
    if (weight_dtype != dtype && weight_dtype != ST_F32)
        return st::fail(ST_ERR_INVALID, "rms_norm: weight dtype %d is neither ST_F32 nor x's, %d", (int)weight_dtype, (int)dtype);
    if (!(eps >= 0.f) || std::isinf(eps)) return st::fail(ST_ERR_INVALID, "rms_norm: eps %g", (double)eps);
    if (rows == 0) return ST_OK;
    if (!x || !weight || (codes != nullptr) != (scales != nullptr)) return st::fail(ST_ERR_INVALID, "rms_norm: NULL buffer (codes and scales go together)");
    if (!y && !codes && !h && !rstd) return st::fail(ST_ERR_INVALID, "rms_norm: no output");
    if (values && !codes) return st::fail(ST_ERR_INVALID, "rms_norm: values without codes");
    const int64_t size = st::dtype_size(dtype);
    if (unaligned(x, size) || unaligned(residual, size) || unaligned(weight, st::dtype_size(weight_dtype)) || unaligned(h, size) || unaligned(y, size) ||
        unaligned(values, size) || unaligned(rstd, 4) || unaligned(scales, 4))
        return st::fail(ST_ERR_INVALID, "rms_norm: a buffer is not aligned to its elements");
    if (!st::device_ok()) return ST_ERR_NO_DEVICE;
    Norm a = {};
    a.x = x, a.residual = residual, a.w = weight, a.rows = rows, a.d = d, a.x_stride = x_stride, a.r_stride = residual_stride, a.eps = eps;
    a.h = h, a.rstd = rstd, a.y = y;
    a.codes = codes, a.c_stride = codes_stride, a.c_width = codes ? std::min(codes_stride, (d + 15) & ~(int64_t)15) : 0;
    a.scales = scales, a.values = values;
    return with_types(dtype, weight_dtype, [&](auto *t, auto *w) -> st_status {
        return launch_rms<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(w)>, true>(a, st::stream_of(stream));
    });
}

extern "C" int64_t st_rms_norm_backward_bytes(int64_t rows, int64_t d, int32_t dtype) {
    if (rows <= 0 || d <= 0 || rows > MOST_ROWS || d > MOST_D) return 0;
    const int64_t parts = back_parts(rows, d, st::dtype_size(dtype));
    return parts > 1 ? parts * d * 4 : 0;
}

extern "C" st_status st_rms_norm_backward(const void *dy, const void *h, const void *dh, int32_t dtype, int64_t rows, int64_t d, int64_t dy_stride,
                                          int64_t h_stride, int64_t dh_stride, const float *rstd, const void *weight, int32_t weight_dtype, void *dx,
                                          float *dweight, void *work, int64_t work_bytes, st_stream stream) {
    st::clear_error();
    if (rows < 0 || d <= 0 || rows > MOST_ROWS || d > MOST_D)
        return st::fail(ST_ERR_INVALID, "rms_norm_backward: rows %lld (up to 2^36), d %lld (1 to 2^30)", (long long)rows, (long long)d);
    if (dy_stride < d || h_stride < d || (dh && dh_stride < d))
        return st::fail(ST_ERR_INVALID, "rms_norm_backward: rows of %lld elements lie %lld, %lld and %lld apart", (long long)d, (long long)dy_stride,
                        (long long)h_stride, (long long)dh_stride);
    if (dtype < ST_F32 || dtype > ST_BF16) return st::fail(ST_ERR_INVALID, "rms_norm_backward: dtype %d is none of ST_F32, ST_F16, ST_BF16", (int)dtype);
    if (weight_dtype != dtype && weight_dtype != ST_F32)
        return st::fail(ST_ERR_INVALID, "rms_norm_backward: weight dtype %d is neither ST_F32 nor the rows', %d", (int)weight_dtype, (int)dtype);
    if (!dweight || (rows && (!dy || !h || !rstd || !weight || !dx))) return st::fail(ST_ERR_INVALID, "rms_norm_backward: NULL buffer");
    const int64_t size = st::dtype_size(dtype), need = st_rms_norm_backward_bytes(rows, d, dtype);
    if (unaligned(dy, size) || unaligned(h, size) || unaligned(dh, size) || unaligned(dx, size) || unaligned(weight, st::dtype_size(weight_dtype)) ||
        unaligned(rstd, 4) || unaligned(dweight, 4) || unaligned(work, 16))
        return st::fail(ST_ERR_INVALID, "rms_norm_backward: a buffer is not aligned to its elements (work: 16 bytes)");
    if (need && (!work || work_bytes < need))
        return st::fail(ST_ERR_INVALID, "rms_norm_backward: %lld bytes of work memory are needed, got %lld", (long long)need, (long long)(work ? work_bytes : 0));
    if (!st::device_ok()) return ST_ERR_NO_DEVICE;
    if (rows == 0) {  // no row: the sum over none
        k_rms_back_sum<<<sum_grid(d), 1024, 0, st::stream_of(stream)>>>(nullptr, 0, d, dweight);
        ST_LAUNCH_CHECK();
        return ST_OK;
    }
    Back a = {};
    a.dy = dy, a.h = h, a.dh = dh, a.w = weight, a.rstd = rstd, a.rows = rows, a.d = d;
    a.dy_stride = dy_stride, a.h_stride = h_stride, a.dh_stride = dh_stride, a.dx = dx, a.part = (float *)work;
    return with_types(dtype, weight_dtype, [&](auto *t, auto *w) -> st_status {
        return launch_back<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(w)>>(a, dweight, st::stream_of(stream));
    });
}
