// Layer norm over the last axis, forward and backward, with the reduction of the weight's and the bias' gradients.
//   mu = mean(x), s = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) s, y = h w + b
//   dx = s (g - mean(g) - h mean(g h)) with g = dy w,  dw = sum over rows of dy h,  db = sum over rows of dy
// Statistics, sums and products in fp32 whatever the storage type; the variance from centred values.
//
// Bound by HBM: each input is read once, each output written once.  A row is held in registers by a group of G lanes (1 .. 64 in
// a wave, 256 or 1024 threads above), ITER vectors of 16 bytes a lane, so statistics and result come from one read.  G is the
// power of two that covers the row: rows of 64 halfs take 8 lanes and a wave works on 8 of them at once (one row per wave would
// leave 7 of 8 lanes idle).  Vectors are loaded and stored at element alignment (global memory takes any), so odd widths,
// strides and addresses go the same way; only the vector that a row's end cuts is taken element by element.
// The backward pass walks rows with the lane's columns fixed: their dw and db sums stay in registers over all rows of a
// workgroup, go through LDS once and to memory as one row of partial sums per workgroup, which a second launch adds in a fixed
// order (no atomics: the same bits for the same inputs).
#include "elem.h"

#include <type_traits>

namespace {

constexpr uint32_t CUS = 256;

// ---- sums over a group of lanes --------------------------------------------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ float dpp(float v)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// every lane of each aligned group of G lanes gets the group's sum, by VALU lane moves alone
template <int G>
__device__ __forceinline__ float lanes_sum(float v)
{
    if constexpr (G >= 2) v += dpp<0xB1>(v);    // quad_perm 1 0 3 2
    if constexpr (G >= 4) v += dpp<0x4E>(v);    // quad_perm 2 3 0 1
    if constexpr (G >= 8) v += dpp<0x141>(v);   // row_half_mirror: the other quad of 8
    if constexpr (G >= 16) v += dpp<0x140>(v);  // row_mirror: the other 8 of 16
    if constexpr (G >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (G >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

// sums of N values over G threads; above a wave through LDS (`turn` alternates between two buffers, so that one barrier is
// enough: a buffer is written again only behind the barrier of the other one)
template <int G, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float *lds, int &turn)
{
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lanes_sum<(G < 64 ? G : 64)>(v[i]);
    if constexpr (G > 64) {
        constexpr int WAVES = G / 64;
        float *mine = lds + turn * (16 * N);
        turn ^= 1;
        const uint32_t wave = threadIdx.x >> 6, first = wave / WAVES * WAVES;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) mine[wave * N + i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = mine[first * N + i];
#pragma unroll
            for (int k = 1; k < WAVES; ++k) s += mine[(first + k) * N + i];
            v[i] = s;
        }
    }
}

// pairwise sum of N values of a lane (N a power of two)
template <int N, class F>
__device__ __forceinline__ float pairwise(F f, int at = 0)
{
    if constexpr (N == 1) return f(at);
    else return pairwise<N / 2>(f, at) + pairwise<N / 2>(f, at + N / 2);
}

// ---- vectors of a row ------------------------------------------------------------------------------------------------------
template <class T> struct Vec16 { static constexpr int N = 16 / sizeof(T); };

template <class T>
__device__ __forceinline__ Vec<T, Vec16<T>::N> load_vec(const T *row, uint32_t col, uint32_t width)
{
    constexpr int N = Vec16<T>::N;
    Vec<T, N> v;
    if (col + N <= width) {
        __builtin_memcpy(&v, row + col, sizeof(v));
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) v.e[k] = (T)0.f;
        if (col < width)
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (col + k < width) v.e[k] = row[col + k];
    }
    return v;
}

template <class T>
__device__ __forceinline__ void store_vec(T *row, uint32_t col, uint32_t width, const Vec<T, Vec16<T>::N> &v)
{
    constexpr int N = Vec16<T>::N;
    if (col + N <= width) {
        __builtin_memcpy(row + col, &v, sizeof(v));
    } else if (col < width) {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (col + k < width) row[col + k] = v.e[k];
    }
}

// N affine parameters from `col` on, fp32 or of the rows' type; `none` where there are none
template <class T, int N>
__device__ __forceinline__ void load_affine(const void *p, bool fp32, uint32_t col, uint32_t width, float none, float (&v)[N])
{
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = none;
    if (!p) return;
    if (fp32) {
        if (col + N <= width) __builtin_memcpy(v, (const float *)p + col, sizeof(v));
        else
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (col + k < width) v[k] = ((const float *)p)[col + k];
    } else {
        const Vec<T, N> t = load_vec((const T *)p, col, width);
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = (float)t.e[k];
    }
}

// ---- forward ---------------------------------------------------------------------------------------------------------------
// U rows of each group are loaded before the first is worked on; a lane's weight and bias stay in registers
template <class T, int G, int ITER, int U>
__global__ void __launch_bounds__(G > 256 ? G : 256)
k_ln_forward(const T *__restrict__ x, uint64_t xs, const void *__restrict__ w, const void *__restrict__ b, int affine_fp32,
             T *__restrict__ y, float *__restrict__ mean, float *__restrict__ rstd, uint64_t rows, uint32_t width,
             float inv_width, float eps)
{
    constexpr int N = Vec16<T>::N, THREADS = G > 256 ? G : 256, GROUPS = THREADS / G;
    __shared__ float lds[G > 64 ? 32 : 1];
    int turn = 0;
    const uint32_t lane = threadIdx.x % G, group = threadIdx.x / G;
    const bool whole = width == (uint32_t)(G * N * ITER);
    float wv[ITER][N], bv[ITER][N];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        load_affine<T>(w, affine_fp32, (i * G + lane) * N, width, 1.f, wv[i]);
        load_affine<T>(b, affine_fp32, (i * G + lane) * N, width, 0.f, bv[i]);
    }
    for (uint64_t tile = blockIdx.x; tile * (GROUPS * U) < rows; tile += gridDim.x) {
        const uint64_t row0 = tile * (GROUPS * U) + group;
        Vec<T, N> raw[U][ITER];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint64_t row = row0 + u * GROUPS;
#pragma unroll
            for (int i = 0; i < ITER; ++i) raw[u][i] = load_vec(x + row * xs, (i * G + lane) * N, row < rows ? width : 0);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint64_t row = row0 + u * GROUPS;
            float v[ITER][N], t[1] = {0.f};
#pragma unroll
            for (int i = 0; i < ITER; ++i) {
#pragma unroll
                for (int k = 0; k < N; ++k) v[i][k] = (float)raw[u][i].e[k];
                t[0] += pairwise<N>([&](int k) { return v[i][k]; });
            }
            group_sum<G>(t, lds, turn);
            const float mu = t[0] * inv_width;
            t[0] = 0.f;
#pragma unroll
            for (int i = 0; i < ITER; ++i) {
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    v[i][k] -= mu;
                    if (!whole && (i * G + lane) * N + k >= width) v[i][k] = 0.f;
                }
                t[0] += pairwise<N>([&](int k) { return v[i][k] * v[i][k]; });
            }
            group_sum<G>(t, lds, turn);
            const float rs = 1.f / sqrtf(t[0] * inv_width + eps);
            if (row < rows) {
#pragma unroll
                for (int i = 0; i < ITER; ++i) {
                    const uint32_t col = (i * G + lane) * N;
                    Vec<T, N> o;
#pragma unroll
                    for (int k = 0; k < N; ++k) o.e[k] = (T)fmaf(v[i][k] * rs, wv[i][k], bv[i][k]);
                    store_vec(y + row * width, col, width, o);
                }
                if (mean && lane == 0) { mean[row] = mu; rstd[row] = rs; }
            }
        }
    }
}

// rows that no workgroup holds in registers: one workgroup of 1024 reads its row three times (from its cache where it fits)
template <class T>
__global__ void __launch_bounds__(1024)
k_ln_forward_long(const T *__restrict__ x, uint64_t xs, const void *__restrict__ w, const void *__restrict__ b, int affine_fp32,
                  T *__restrict__ y, float *__restrict__ mean, float *__restrict__ rstd, uint64_t rows, uint32_t width,
                  float inv_width, float eps)
{
    constexpr int N = Vec16<T>::N;
    __shared__ float lds[32];
    int turn = 0;
    for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * xs;
        float t[1] = {0.f};
        for (uint64_t c = threadIdx.x * N; c < width; c += 1024 * N) {
            const Vec<T, N> v = load_vec(xr, (uint32_t)c, width);
            t[0] += pairwise<N>([&](int k) { return (float)v.e[k]; });
        }
        group_sum<1024>(t, lds, turn);
        const float mu = t[0] * inv_width;
        t[0] = 0.f;
        for (uint64_t c = threadIdx.x * N; c < width; c += 1024 * N) {
            const Vec<T, N> v = load_vec(xr, (uint32_t)c, width);
            t[0] += pairwise<N>([&](int k) { const float d = c + k < width ? (float)v.e[k] - mu : 0.f; return d * d; });
        }
        group_sum<1024>(t, lds, turn);
        const float rs = 1.f / sqrtf(t[0] * inv_width + eps);
        for (uint64_t c = threadIdx.x * N; c < width; c += 1024 * N) {
            Vec<T, N> v = load_vec(xr, (uint32_t)c, width);
            float wv[N], bv[N];
            load_affine<T>(w, affine_fp32, (uint32_t)c, width, 1.f, wv);
            load_affine<T>(b, affine_fp32, (uint32_t)c, width, 0.f, bv);
#pragma unroll
            for (int k = 0; k < N; ++k) v.e[k] = (T)fmaf(((float)v.e[k] - mu) * rs, wv[k], bv[k]);
            store_vec(y + row * width, (uint32_t)c, width, v);
        }
        if (mean && threadIdx.x == 0) { mean[row] = mu; rstd[row] = rs; }
    }
}

// ---- backward --------------------------------------------------------------------------------------------------------------
constexpr int BWD_THREADS = 1024;

template <class W> __device__ __forceinline__ void put_column(void *p, uint32_t col, float v) { ((W *)p)[col] = (W)v; }

// sums of a workgroup's rows for its columns: one workgroup alone stores the results, of several each stores a row of partial
// sums [2][width]
template <class T>
__device__ __forceinline__ void store_sum(int which, uint32_t col, float v, uint32_t width, float *part, void *dw, void *db, int affine_fp32)
{
    if (gridDim.x > 1) {
        part[((uint64_t)blockIdx.x * 2 + which) * width + col] = v;
    } else if (void *p = which ? db : dw) {
        affine_fp32 ? put_column<float>(p, col, v) : put_column<T>(p, col, v);
    }
}

template <class T, int G, int ITER, int U>
__global__ void __launch_bounds__(BWD_THREADS)
k_ln_backward(const T *__restrict__ dy, uint64_t dys, const T *__restrict__ x, uint64_t xs, const void *__restrict__ w,
              int affine_fp32, const float *__restrict__ mean, const float *__restrict__ rstd, T *__restrict__ dx, void *dw,
              void *db, float *__restrict__ part, uint64_t rows, uint32_t width, float inv_width)
{
    constexpr int N = Vec16<T>::N, GROUPS = BWD_THREADS / G;
    // sums: the groups of a wave are added by lane moves first, so LDS holds one row of G ITER N columns per wave or group
    constexpr int SETS = G < 64 ? BWD_THREADS / 64 : GROUPS;
    __shared__ float lds[G > 64 ? 64 : 1];
    __shared__ float sums[SETS > 1 ? SETS * G * N : 1];
    int turn = 0;
    const uint32_t lane = threadIdx.x % G, group = threadIdx.x / G;
    float wv[ITER][N], sw[ITER][N], sb[ITER][N];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        load_affine<T>(w, affine_fp32, (i * G + lane) * N, width, 1.f, wv[i]);
#pragma unroll
        for (int k = 0; k < N; ++k) sw[i][k] = sb[i][k] = 0.f;
    }
    for (uint64_t tile = blockIdx.x; tile * (GROUPS * U) < rows; tile += gridDim.x) {
        const uint64_t row0 = tile * (GROUPS * U) + group;
        Vec<T, N> xr[U][ITER], dr[U][ITER];
        float mu[U], rs[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint64_t row = row0 + u * GROUPS;
            const uint32_t live = row < rows ? width : 0;  // (what lies outside is zero: it adds nothing to any sum)
#pragma unroll
            for (int i = 0; i < ITER; ++i) {
                xr[u][i] = load_vec(x + row * xs, (i * G + lane) * N, live);
                dr[u][i] = load_vec(dy + row * dys, (i * G + lane) * N, live);
            }
            mu[u] = live ? mean[row] : 0.f;
            rs[u] = live ? rstd[row] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint64_t row = row0 + u * GROUPS;
            float h[ITER][N], g[ITER][N], t[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < ITER; ++i) {
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    const float d = (float)dr[u][i].e[k];
                    h[i][k] = ((float)xr[u][i].e[k] - mu[u]) * rs[u];
                    g[i][k] = d * wv[i][k];
                    sw[i][k] = fmaf(d, h[i][k], sw[i][k]);
                    sb[i][k] += d;
                }
                t[0] += pairwise<N>([&](int k) { return g[i][k]; });
                t[1] += pairwise<N>([&](int k) { return g[i][k] * h[i][k]; });
            }
            if (dx) {  // (the same for every thread)
                group_sum<G>(t, lds, turn);
                const float a = t[0] * inv_width, c = t[1] * inv_width;
                if (row < rows)
#pragma unroll
                    for (int i = 0; i < ITER; ++i) {
                        Vec<T, N> o;
#pragma unroll
                        for (int k = 0; k < N; ++k) o.e[k] = (T)(rs[u] * (g[i][k] - a - h[i][k] * c));
                        store_vec(dx + row * width, (i * G + lane) * N, width, o);
                    }
            }
        }
    }
    if (!dw && !db) return;
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            float(&s)[N] = which ? sb[i] : sw[i];
            if constexpr (SETS == 1) {
#pragma unroll
                for (int k = 0; k < N; ++k)
                    if ((i * G + lane) * N + k < width) store_sum<T>(which, (i * G + lane) * N + k, s[k], width, part, dw, db, affine_fp32);
            } else {
#pragma unroll
                for (int k = 0; k < N; ++k)
#pragma unroll
                    for (int o = G; o < 64; o <<= 1) s[k] += __shfl_xor(s[k], o, 64);
                __syncthreads();
                const uint32_t set = G < 64 ? threadIdx.x >> 6 : group;
                if (G >= 64 || (threadIdx.x & 63) < G)
#pragma unroll
                    for (int k = 0; k < N; ++k) sums[(set * N + k) * G + lane] = s[k];
                __syncthreads();
                for (uint32_t c = threadIdx.x; c < (uint32_t)(G * N); c += BWD_THREADS) {  // c = k G + lane
                    const uint32_t col = (i * G + c % G) * N + c / G;
                    float v = sums[c];
                    for (int q = 1; q < SETS; ++q) v += sums[q * (G * N) + c];
                    if (col < width) store_sum<T>(which, col, v, width, part, dw, db, affine_fp32);
                }
            }
        }
}

// long rows: dx alone, one workgroup per row, two reads
template <class T>
__global__ void __launch_bounds__(BWD_THREADS)
k_ln_backward_long_rows(const T *__restrict__ dy, uint64_t dys, const T *__restrict__ x, uint64_t xs, const void *__restrict__ w,
                        int affine_fp32, const float *__restrict__ mean, const float *__restrict__ rstd, T *__restrict__ dx,
                        uint64_t rows, uint32_t width, float inv_width)
{
    constexpr int N = Vec16<T>::N;
    __shared__ float lds[64];
    int turn = 0;
    for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * xs, *dr = dy + row * dys;
        const float mu = mean[row], rs = rstd[row];
        float t[2] = {0.f, 0.f};
        for (int pass = 0; pass < 2; ++pass) {
            const float a = t[0] * inv_width, c = t[1] * inv_width;
            for (uint64_t at = threadIdx.x * N; at < width; at += BWD_THREADS * N) {
                const Vec<T, N> xv = load_vec(xr, (uint32_t)at, width), dv = load_vec(dr, (uint32_t)at, width);
                float wv[N], h[N], g[N];
                load_affine<T>(w, affine_fp32, (uint32_t)at, width, 1.f, wv);
#pragma unroll
                for (int k = 0; k < N; ++k) { h[k] = ((float)xv.e[k] - mu) * rs; g[k] = (float)dv.e[k] * wv[k]; }
                if (pass == 0) {
                    t[0] += pairwise<N>([&](int k) { return g[k]; });
                    t[1] += pairwise<N>([&](int k) { return g[k] * h[k]; });
                } else {
                    Vec<T, N> o;
#pragma unroll
                    for (int k = 0; k < N; ++k) o.e[k] = (T)(rs * (g[k] - a - h[k] * c));
                    store_vec(dx + row * width, (uint32_t)at, width, o);
                }
            }
            if (pass == 0) group_sum<BWD_THREADS>(t, lds, turn);
        }
    }
}

// long rows: dw and db alone, a workgroup for 1024 N columns (blockIdx.y) of some of the rows (blockIdx.x)
template <class T>
__global__ void __launch_bounds__(BWD_THREADS)
k_ln_backward_long_columns(const T *__restrict__ dy, uint64_t dys, const T *__restrict__ x, uint64_t xs,
                           const float *__restrict__ mean, const float *__restrict__ rstd, float *__restrict__ part, void *dw,
                           void *db, int affine_fp32, uint64_t rows, uint32_t width)
{
    constexpr int N = Vec16<T>::N;
    const uint64_t col = ((uint64_t)blockIdx.y * BWD_THREADS + threadIdx.x) * N;
    if (col >= width) return;
    float sw[N] = {}, sb[N] = {};
    for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const Vec<T, N> xv = load_vec(x + row * xs, (uint32_t)col, width), dv = load_vec(dy + row * dys, (uint32_t)col, width);
        const float mu = mean[row], rs = rstd[row];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            sw[k] = fmaf((float)dv.e[k], ((float)xv.e[k] - mu) * rs, sw[k]);
            sb[k] += (float)dv.e[k];
        }
    }
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (col + k < width) {
            store_sum<T>(0, (uint32_t)col + k, sw[k], width, part, dw, db, affine_fp32);
            store_sum<T>(1, (uint32_t)col + k, sb[k], width, part, dw, db, affine_fp32);
        }
}

// the workgroups' partial sums [n][2 width] of 16 columns, 64 of them at a time; n = 0: no rows
template <class T>
__global__ void __launch_bounds__(1024)
k_ln_backward_finish(const float *__restrict__ part, uint32_t n, uint32_t width, void *dw, void *db, int affine_fp32)
{
    const uint64_t col = (uint64_t)blockIdx.x * 16 + threadIdx.x % 16;
    float acc = 0.f;
    if (col < 2ull * width)
#pragma unroll 8
        for (uint32_t s = threadIdx.x / 16; s < n; s += 64) acc += part[s * 2ull * width + col];
    acc += __shfl_xor(acc, 16, 64);
    acc += __shfl_xor(acc, 32, 64);
    __shared__ float sums[16][16];
    if ((threadIdx.x & 63) < 16) sums[threadIdx.x >> 6][threadIdx.x & 15] = acc;
    __syncthreads();
    if (threadIdx.x >= 16 || col >= 2ull * width) return;
    float v = sums[0][threadIdx.x];
    for (int q = 1; q < 16; ++q) v += sums[q][threadIdx.x];
    void *p = col < width ? dw : db;
    const uint32_t c = (uint32_t)(col < width ? col : col - width);
    if (p) affine_fp32 ? put_column<float>(p, c, v) : put_column<T>(p, c, v);
}

// ---- host ------------------------------------------------------------------------------------------------------------------
template <int V> using Int = std::integral_constant<int, V>;

template <class F>
int ln_type(uint32_t dtype, F f)
{
    if (dtype == DT_F32) return f(float{});
    if (dtype == DT_F16) return f(_Float16{});
    return f(__bf16{});
}

bool misaligned(const void *p, uint32_t dtype) { return ((uintptr_t)p & (dtype_size(dtype) - 1)) != 0; }

int ln_check(const char *what, uint64_t rows, uint32_t width, uint32_t dtype, uint32_t affine)
{
    NSR_REQUIRE(width >= 1 && width <= (1u << 30), "%s: width %u (1 .. 2^30)", what, width);
    NSR_REQUIRE(rows < (1ull << 40), "%s: 2^40 rows or more", what);
    NSR_REQUIRE(dtype <= DT_BF16, "%s: dtype %u (0 fp32, 1 fp16, 2 bf16)", what, dtype);
    NSR_REQUIRE(affine == DT_F32 || affine == dtype, "%s: weight and bias are fp32 or of the input's type", what);
    return NSR_OK;
}

// the group size for rows of `width` elements of n per vector, up to a wave: f(G)
template <int N, class F>
int narrow_group(uint32_t width, F f)
{
    const uint32_t vectors = nsr_div_up(width, N);
    if (vectors <= 1) return f(Int<1>{});
    if (vectors <= 2) return f(Int<2>{});
    if (vectors <= 4) return f(Int<4>{});
    if (vectors <= 8) return f(Int<8>{});
    if (vectors <= 16) return f(Int<16>{});
    if (vectors <= 32) return f(Int<32>{});
    return f(Int<64>{});
}

// f(G, ITER): at most 16 columns a lane in the forward pass.  In the backward pass each column has a weight, two sums and two
// inputs in registers: 16 in groups of up to 256, 8 where 1024 threads share the registers of a CU.
constexpr uint32_t FORWARD_MOST = 16384, BACKWARD_MOST = 8192;

template <class T, uint32_t MOST, class F>
int row_shape(uint32_t width, F f)
{
    constexpr uint32_t N = Vec16<T>::N;
    if (width <= 64 * N) return narrow_group<(int)N>(width, [&](auto g) { return f(g, Int<1>{}); });
    if (width <= 128 * N) return f(Int<64>{}, Int<2>{});
    if (width <= 256 * N) return f(Int<256>{}, Int<1>{});
    if (width <= 512 * N) return f(Int<256>{}, Int<2>{});
    if constexpr (MOST >= 1024 * N)
        if (width <= 1024 * N) return f(Int<1024>{}, Int<1>{});
    if constexpr (MOST >= 2048 * N)
        if (width <= 2048 * N) return f(Int<1024>{}, Int<2>{});
    return f(Int<1024>{}, Int<MOST / (1024 * N)>{});
}

// rows of each group that are in flight at once
constexpr int rows_at_once(int iter) { return iter == 1 ? 2 : 1; }

// workgroups of the backward pass = rows of partial sums
uint32_t backward_groups(uint64_t rows, uint32_t width, uint32_t dtype)
{
    if (rows == 0) return 0;
    uint64_t per = 1;
    if (width <= BACKWARD_MOST)
        ln_type(dtype, [&](auto t) {
            return row_shape<decltype(t), BACKWARD_MOST>(width, [&](auto g, auto iter) {
                per = BWD_THREADS / decltype(g)::value * rows_at_once(decltype(iter)::value);
                return 0;
            });
        });
    const uint64_t tiles = (rows + per - 1) / per, most = 2 * CUS;
    return (uint32_t)(tiles < most ? tiles : most);
}

}  // namespace

extern "C" int nsr_layer_norm_forward(const void *x, uint64_t x_stride, const void *weight, const void *bias, void *y,
                                      float *mean, float *rstd, uint64_t rows, uint32_t width, uint32_t dtype,
                                      uint32_t affine_dtype, float eps, void *stream)
{
    const int rc = ln_check("nsr_layer_norm_forward", rows, width, dtype, affine_dtype);
    if (rc != NSR_OK) return rc;
    NSR_REQUIRE(eps >= 0.f, "nsr_layer_norm_forward: eps >= 0");
    NSR_REQUIRE((mean == nullptr) == (rstd == nullptr), "nsr_layer_norm_forward: mean and rstd come together");
    if (rows == 0) return NSR_OK;
    NSR_REQUIRE(x && y, "nsr_layer_norm_forward: NULL pointer");
    NSR_REQUIRE(x_stride >= width || rows == 1, "nsr_layer_norm_forward: rows overlap");
    NSR_REQUIRE(!misaligned(x, dtype) && !misaligned(y, dtype) && !misaligned(weight, affine_dtype) &&
                    !misaligned(bias, affine_dtype) && (((uintptr_t)mean | (uintptr_t)rstd) & 3) == 0,
                "nsr_layer_norm_forward: misaligned pointer");
    const int fp32 = affine_dtype == DT_F32;
    const float inv = 1.f / (float)width;
    return ln_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (width > FORWARD_MOST) {
            hipLaunchKernelGGL((k_ln_forward_long<T>), dim3(rows < 4 * CUS ? (uint32_t)rows : 4 * CUS), dim3(1024), 0,
                               (hipStream_t)stream, (const T *)x, x_stride, weight, bias, fp32, (T *)y, mean, rstd, rows, width,
                               inv, eps);
            NSR_CHECK_LAUNCH("nsr_layer_norm_forward");
            return NSR_OK;
        }
        return row_shape<T, FORWARD_MOST>(width, [&](auto g, auto iter) {
            constexpr int G = decltype(g)::value, ITER = decltype(iter)::value, U = rows_at_once(ITER);
            constexpr int THREADS = G > 256 ? G : 256;
            const uint64_t tiles = (rows + THREADS / G * U - 1) / (THREADS / G * U), most = 8 * CUS * 256 / THREADS;
            hipLaunchKernelGGL((k_ln_forward<T, G, ITER, U>), dim3((uint32_t)(tiles < most ? tiles : most)), dim3(THREADS), 0,
                               (hipStream_t)stream, (const T *)x, x_stride, weight, bias, fp32, (T *)y, mean, rstd, rows, width,
                               inv, eps);
            NSR_CHECK_LAUNCH("nsr_layer_norm_forward");
            return NSR_OK;
        });
    });
}

extern "C" uint64_t nsr_layer_norm_backward_workspace_floats(uint64_t rows, uint32_t width, uint32_t dtype)
{
    if (width == 0 || dtype > DT_BF16) return 0;
    const uint32_t n = backward_groups(rows, width, dtype);
    return n > 1 ? (uint64_t)n * 2 * width : 0;
}

extern "C" int nsr_layer_norm_backward(const void *dy, uint64_t dy_stride, const void *x, uint64_t x_stride, const void *weight,
                                       const float *mean, const float *rstd, void *dx, void *dweight, void *dbias,
                                       float *workspace, uint64_t rows, uint32_t width, uint32_t dtype, uint32_t affine_dtype,
                                       void *stream)
{
    const int rc = ln_check("nsr_layer_norm_backward", rows, width, dtype, affine_dtype);
    if (rc != NSR_OK) return rc;
    const bool affine = dweight || dbias;
    const uint32_t groups = backward_groups(rows, width, dtype);
    NSR_REQUIRE(rows == 0 || (dy && x && mean && rstd), "nsr_layer_norm_backward: NULL pointer");
    NSR_REQUIRE(groups <= 1 || !affine || workspace, "nsr_layer_norm_backward: the affine gradients need the workspace");
    NSR_REQUIRE((x_stride >= width && dy_stride >= width) || rows <= 1, "nsr_layer_norm_backward: rows overlap");
    NSR_REQUIRE(!misaligned(dy, dtype) && !misaligned(x, dtype) && !misaligned(dx, dtype) && !misaligned(weight, affine_dtype) &&
                    !misaligned(dweight, affine_dtype) && !misaligned(dbias, affine_dtype) &&
                    (((uintptr_t)workspace | (uintptr_t)mean | (uintptr_t)rstd) & 3) == 0,
                "nsr_layer_norm_backward: misaligned pointer");
    if (!affine && !(dx && rows)) return NSR_OK;
    const int fp32 = affine_dtype == DT_F32;
    const float inv = 1.f / (float)width;
    hipStream_t st = (hipStream_t)stream;
    return ln_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (groups && width <= BACKWARD_MOST) {
            row_shape<T, BACKWARD_MOST>(width, [&](auto g, auto iter) {
                constexpr int G = decltype(g)::value, ITER = decltype(iter)::value;
                hipLaunchKernelGGL((k_ln_backward<T, G, ITER, rows_at_once(ITER)>), dim3(groups), dim3(BWD_THREADS), 0, st,
                                   (const T *)dy, dy_stride, (const T *)x, x_stride, weight, fp32, mean, rstd, (T *)dx, dweight,
                                   dbias, workspace, rows, width, inv);
                return 0;
            });
        } else if (groups) {
            if (dx)
                hipLaunchKernelGGL((k_ln_backward_long_rows<T>), dim3(rows < 4 * CUS ? (uint32_t)rows : 4 * CUS), dim3(BWD_THREADS),
                                   0, st, (const T *)dy, dy_stride, (const T *)x, x_stride, weight, fp32, mean, rstd, (T *)dx, rows,
                                   width, inv);
            if (affine)
                hipLaunchKernelGGL((k_ln_backward_long_columns<T>), dim3(groups, nsr_div_up(width, BWD_THREADS * Vec16<T>::N)),
                                   dim3(BWD_THREADS), 0, st, (const T *)dy, dy_stride, (const T *)x, x_stride, mean, rstd,
                                   workspace, dweight, dbias, fp32, rows, width);
        }
        if (affine && groups != 1)
            hipLaunchKernelGGL((k_ln_backward_finish<T>), dim3(nsr_div_up(2ull * width, 16)), dim3(1024), 0, st, workspace, groups,
                               width, dweight, dbias, fp32);
        NSR_CHECK_LAUNCH("nsr_layer_norm_backward");
        return NSR_OK;
    });
}
