// Layer norm over the last axis, forward and backward, with the reduction of the weight's and the bias' gradients.
//   mu = mean(x), s = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) s, y = h w + b
//   dx = s (g - mean(g) - h mean(g h)) with g = dy w,  dw = sum over rows of dy h,  db = sum over rows of dy
// Statistics, sums and products in fp32 whatever the storage type; the variance from centred values.
//
// Bound by HBM: each input is read once, each output written once.  A row is held in registers by a group of G lanes, ITER
// vectors of 16 bytes a lane, so statistics and result come from one read.  G is the power of two that covers the row, 1 .. 64
// lanes of a wave, 128 .. 1024 threads above: rows of 64 halfs take 8 lanes and a wave works on 8 of them at once (one row per
// wave would leave 7 of 8 lanes idle).  Odd widths: the vector at a row's end starts early enough to be whole, what it repeats
// of the one before counts in no sum and is stored twice with the same value.
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

// sums of N values (1 or 2) over G threads.  Two values share the way: a swap of half groups leaves the one's partial sums in the
// lower half and the other's in the upper, so that one register goes through the rest.  Above a wave through LDS (`turn` alternates
// between two buffers, so that one barrier is enough: a buffer is written again only behind the barrier of the other one), where a
// lane reads one wave's sum and lane moves add them.
template <int G, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float *lds, int &turn)
{
    static_assert(N == 1 || N == 2, "one value or two");
    constexpr bool HALVES = N == 2 && G >= 32;
    constexpr int HALF = G == 32 ? 16 : 32;
    auto swapped = [](float a, float b) {
        if constexpr (G == 32) return __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
        else return __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    };
    if constexpr (HALVES) {
        const auto r = swapped(v[0], v[N - 1]);
        v[0] = lanes_sum<HALF>(__uint_as_float(r[0]) + __uint_as_float(r[1]));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = lanes_sum<(G < 64 ? G : 64)>(v[i]);
    }
    if constexpr (G > 64) {
        constexpr int WAVES = G / 64, LANES = 64 / N;  // (lanes that hold the same value)
        float *mine = lds + turn * (16 * N);
        turn ^= 1;
        const uint32_t wave = threadIdx.x >> 6, which = N == 1 ? 0 : threadIdx.x >> 5 & 1, first = wave / WAVES * WAVES;
        if (threadIdx.x % LANES == 0) mine[wave * N + which] = v[0];
        __syncthreads();
        v[0] = lanes_sum<WAVES>(mine[(first + threadIdx.x % WAVES) * N + which]);
    }
    if constexpr (HALVES) {
        const auto r = swapped(v[0], v[0]);
        v[0] = __uint_as_float(r[0]);
        v[N - 1] = __uint_as_float(r[1]);
    }
}

// pairwise sum of N values of a lane (N a power of two)
template <int N, class F>
__device__ __forceinline__ float pairwise(F f, int at = 0)
{
    if constexpr (N == 1) return f(at);
    else return pairwise<N / 2>(f, at) + pairwise<N / 2>(f, at + N / 2);
}

// 1 / sqrt(v) to 1 ulp; the instruction takes denormal numbers for zero
__device__ __forceinline__ float inverse_sqrt(float v)
{
    const bool small = v < 0x1p-100f;
    return __builtin_amdgcn_rsqf(small ? v * 0x1p100f : v) * (small ? 0x1p50f : 1.f);
}

// t / n, rounded as the division is: one step from t times the rounded 1 / n.  (sum times 1 / n alone misses the mean of a constant
// row by an ulp at every fourth width: 0.02 of the centred value 0 for rows of 1000 and an eps of 1e-5.)
__device__ __forceinline__ float quotient(float t, float n, float inv_n)
{
    const float q = t * inv_n;
    return __builtin_amdgcn_div_fixupf(fmaf(fmaf(-q, n, t), inv_n, q), n, t);  // (of infinities and NaN)
}

// What the centred values v = x - mu of a row still sum up to is the error of mu, an ulp or more of it where the sum was rounded:
// their mean `off` goes with the squares' sum through one reduction, and what follows takes the mean as mu + off.  So a mean far
// above the spread costs rounding of the inputs' differences alone.
struct Statistics { float off, rstd; };
__device__ __forceinline__ Statistics row_statistics(float squares, float sum, float inv_n, float eps)
{
    const float off = sum * inv_n, about = squares * inv_n;
    // (the difference is under 0 by rounding alone; squares past fp32, where off's may be too, leave 1 / sqrt at 0, and NaN stays)
    const float var = about < __builtin_inff() ? fmaxf(fmaf(-off, off, about), 0.f) : about;
    return {off, inverse_sqrt(var + eps)};
}

// sum of f(k) g(k), k < N, in two chains of fma
template <int N, class F, class H>
__device__ __forceinline__ float dot(F f, H g)
{
    float a = f(0) * g(0), b = N > 1 ? f(1 % N) * g(1 % N) : 0.f;
#pragma unroll
    for (int k = 2; k < N; k += 2) {
        a = fmaf(f(k), g(k), a);
        b = fmaf(f(k + 1), g(k + 1), b);
    }
    return a + b;
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

// How a row's vectors are read and written:
//   BUFFER  rows at 4-byte addresses (fp32; 16 bits with even widths and strides): buffer instructions, where lanes outside the
//           row and rows past the end have offsets past the buffer's end: loads give zero, stores do nothing;
//   GLOBAL  16-bit rows at odd addresses: global instructions, which take any address; a lane outside the row repeats its last
//           vector and a row past the end the last row, and neither stores;
//   TINY    rows of less than a vector, element by element.
// In the first two nothing branches around a load, in the first around a store either, and only so can the compiler count what
// is outstanding: behind a branch it waits for everything, also for the loads of the next row and the stores of the last one
// (backward, 131072 x 256 bf16: 47.7 us with branches, 41.8 without; 516222 x 65 bf16: 89.9 and 55.4 us).
enum Access { BUFFER, GLOBAL, TINY };
constexpr uint32_t OUTSIDE = 0x80000000u, BUFFER_MOST = 0x7ffffff0u;

// `left` rows of `row_bytes`, `stride_bytes` apart, from p on (the same values in every lane)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_buffer(const void *p, int64_t left, uint64_t stride_bytes, uint32_t row_bytes)
{
    const uint64_t bytes = left > 0 ? (uint64_t)(left - 1) * stride_bytes + row_bytes : 0;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, (int)(bytes < BUFFER_MOST ? bytes : BUFFER_MOST), 0x00020000);
}

template <class V>
__device__ __forceinline__ V buffer_load(__amdgpu_buffer_rsrc_t r, uint32_t offset)
{
    V v;
    if constexpr (sizeof(V) == 16) {
        const auto u = __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, 0);
        __builtin_memcpy(&v, &u, 16);
    } else {
        const auto u = __builtin_amdgcn_raw_buffer_load_b32(r, offset, 0, 0);
        __builtin_memcpy(&v, &u, 4);
    }
    return v;
}

template <class V>
__device__ __forceinline__ void buffer_store(__amdgpu_buffer_rsrc_t r, uint32_t offset, const V &v)
{
    if constexpr (sizeof(V) == 16) {
        decltype(__builtin_amdgcn_raw_buffer_load_b128(r, 0, 0, 0)) u;
        __builtin_memcpy(&u, &v, 16);
        __builtin_amdgcn_raw_buffer_store_b128(u, r, offset, 0, 0);
    } else {
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), r, offset, 0, 0);
    }
}

// where a vector of the row lies: its first column, and how many of its elements the vector before holds too (all of them, or
// more: a lane outside the row)
struct Place { uint32_t at, twice; };
template <int N, Access A>
__device__ __forceinline__ Place place(uint32_t vector, uint32_t width)
{
    const uint32_t col = vector * N;
    if constexpr (A == TINY) return {col, 0};
    const uint32_t at = col + N <= width ? col : width - N;
    return {at, col - at};
}

// the rows of a tile, row0 .. row0 + GROUPS - 1, in memory; group_at = group * stride
template <class T, Access A, int GROUPS>
struct Rows {
    static constexpr int N = Vec16<T>::N;
    __amdgpu_buffer_rsrc_t buffer;
    T *row;
    uint32_t at0, width;  // (width 0: nothing to write, nor to read where the access is TINY)

    __device__ __forceinline__ Rows(const T *p, uint64_t stride, uint64_t row0, uint32_t group, uint64_t group_at, uint64_t rows,
                                    uint32_t width_) : width(width_)
    {
        if constexpr (A == BUFFER) {
            buffer = rows_buffer(p + row0 * stride, (int64_t)(rows - row0), stride * sizeof(T), width_ * sizeof(T));
            at0 = (uint32_t)group_at;
        } else {
            const uint64_t r0 = row0 < rows ? row0 : rows - 1;  // (the same in every lane)
            row = const_cast<T *>(p) + r0 * stride;
            if constexpr (GROUPS > 1) {
                const uint64_t last = rows - 1 - r0;
                if (last >= GROUPS - 1) row += group_at;
                else row += (group < last ? group : last) * stride;
                if (row0 + group >= rows) width = 0;
            }
        }
    }
    __device__ __forceinline__ Vec<T, N> load(const Place &p) const
    {
        if constexpr (A == BUFFER) return buffer_load<Vec<T, N>>(buffer, p.twice < N ? (at0 + p.at) * sizeof(T) : OUTSIDE);
        if constexpr (A == TINY) return load_vec(row, p.at, width);
        Vec<T, N> v;
        __builtin_memcpy(&v, row + p.at, sizeof(v));
        return v;
    }
    __device__ __forceinline__ void store(const Place &p, const Vec<T, N> &v) const
    {
        if constexpr (A == BUFFER) buffer_store(buffer, p.twice < N ? (at0 + p.at) * sizeof(T) : OUTSIDE, v);
        else if constexpr (A == TINY) store_vec(row, p.at, width, v);
        else if (p.twice < N && (GROUPS == 1 || width)) __builtin_memcpy(row + p.at, &v, sizeof(v));
    }
};

// the vector, or zeros
template <class V>
__device__ __forceinline__ V kept(V v, bool keep)
{
    uint32_t u[sizeof(V) / 4];
    __builtin_memcpy(u, &v, sizeof(v));
#pragma unroll
    for (uint32_t &w : u) w = keep ? w : 0u;
    __builtin_memcpy(&v, u, sizeof(v));
    return v;
}

// N affine parameters from `col` on, fp32 or of the rows' type; `none` where there are none.  WHOLE: all N are in the row
template <class T, bool WHOLE, int N>
__device__ __forceinline__ void load_affine(const void *p, bool fp32, uint32_t col, uint32_t width, float none, float (&v)[N])
{
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = none;
    if (!p) return;
    if (fp32) {
        if (WHOLE || col + N <= width) __builtin_memcpy(v, (const float *)p + col, sizeof(v));
        else
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (col + k < width) v[k] = ((const float *)p)[col + k];
    } else {
        Vec<T, N> t;
        if constexpr (WHOLE) __builtin_memcpy(&t, (const T *)p + col, sizeof(t));
        else t = load_vec((const T *)p, col, width);
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = (float)t.e[k];
    }
}

// ---- forward ---------------------------------------------------------------------------------------------------------------
// Two reductions over the row's registers (mean; squares and what is left of the sum about it), two fma an element with weight
// and bias, which stay in registers.  Bound by HBM: 2097152 x 64 fp16 in 94 us (5.7 TB/s), 8192 x 4096 bf16 in 24 us (5.6 TB/s).
// Groups of more than a wave load the next row while they work on one; smaller ones have enough waves without (2097152 x 64 fp16:
// 94 us without, 101 us with).  16-bit rows that leave lanes of their group idle are bound by the vector units beside (16376 x 2049
// bf16 32 us, 6709 x 5001 32 us; with every lane's elements masked 40 and 42 us).
template <class T, int G, int ITER, Access A>
__global__ void __launch_bounds__(G > 256 ? G : 256)
k_ln_forward(const T *__restrict__ x, uint64_t xs, const void *__restrict__ w, const void *__restrict__ b, int affine_fp32,
             T *__restrict__ y, float *__restrict__ mean, float *__restrict__ rstd, uint64_t rows, uint32_t width,
             float inv_width, float eps)
{
    constexpr int N = Vec16<T>::N, THREADS = G > 256 ? G : 256, GROUPS = THREADS / G;
    __shared__ float lds[G > 64 ? 64 : 1];
    int turn = 0;
    const float n = (float)width;
    const uint32_t lane = threadIdx.x % G, group = threadIdx.x / G;
    const uint64_t x_at = group * xs, y_at = (uint64_t)group * width;
    Vec<T, N> raw[ITER];
    auto load_row = [&](uint64_t tile) {
        const Rows<T, A, GROUPS> from(x, xs, tile * GROUPS, group, x_at, rows, width);
#pragma unroll
        for (int i = 0; i < ITER; ++i) raw[i] = from.load(place<N, A>(i * G + lane, width));
    };
    load_row(blockIdx.x);
    float wv[ITER][N], bv[ITER][N];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const Place p = place<N, A>(i * G + lane, width);
        load_affine<T, A != TINY>(w, affine_fp32, p.at, width, 1.f, wv[i]);
        load_affine<T, A != TINY>(b, affine_fp32, p.at, width, 0.f, bv[i]);
    }
    // 1 where element k of vector i counts in the sums.  A group is the smallest that covers the row, so the first half of a lane's
    // vectors is whole, and of the rest that of most waves above one a row: nothing is masked there.
    constexpr int FIRST = ITER / 2;
    float mask[ITER - FIRST][N];
    bool all = true;
#pragma unroll
    for (int i = FIRST; i < ITER; ++i) {
        const Place p = place<N, A>(i * G + lane, width);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const bool counts = A == TINY ? p.at + k < width : k >= (int)p.twice;
            mask[i - FIRST][k] = counts ? 1.f : 0.f;
            all = all && counts;
        }
    }
    const bool whole = __all(all);
    for (uint64_t tile = blockIdx.x; tile * GROUPS < rows; tile += gridDim.x) {
        const uint64_t row0 = tile * GROUPS;
        const int64_t left = mean ? (int64_t)(rows - row0) : 0;  // (of the statistics)
        float v[ITER][N], t[1] = {0.f};
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
#pragma unroll
            for (int k = 0; k < N; ++k) v[i][k] = (float)raw[i].e[k];
            if (i < FIRST || whole) t[0] += pairwise<N>([&](int k) { return v[i][k]; });
            else t[0] += dot<N>([&](int k) { return v[i][k]; }, [&](int k) { return mask[i - FIRST][k]; });
        }
        if constexpr (G > 64) load_row(tile + gridDim.x);
        group_sum<G>(t, lds, turn);
        const float mu = quotient(t[0], n, inv_width);
        float c[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
#pragma unroll
            for (int k = 0; k < N; ++k) v[i][k] -= mu;
            if (i < FIRST || whole) {
                c[0] += dot<N>([&](int k) { return v[i][k]; }, [&](int k) { return v[i][k]; });
                c[1] += pairwise<N>([&](int k) { return v[i][k]; });
            } else {
                float once[N];
#pragma unroll
                for (int k = 0; k < N; ++k) once[k] = v[i][k] * mask[i - FIRST][k];
                c[0] += dot<N>([&](int k) { return once[k]; }, [&](int k) { return v[i][k]; });
                c[1] += pairwise<N>([&](int k) { return once[k]; });
            }
        }
        group_sum<G>(c, lds, turn);
        const Statistics st = row_statistics(c[0], c[1], inv_width, eps);
        const float rs = st.rstd, shift = -st.off * rs;
        const Rows<T, A, GROUPS> to(y, width, row0, group, y_at, rows, width);
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            Vec<T, N> o;
#pragma unroll
            for (int k = 0; k < N; ++k) o.e[k] = (T)fmaf(fmaf(v[i][k], rs, shift), wv[i][k], bv[i][k]);
            to.store(place<N, A>(i * G + lane, width), o);
        }
        buffer_store(rows_buffer(mean + row0, left, 4, 4), lane == 0 ? group * 4 : OUTSIDE, mu + st.off);
        buffer_store(rows_buffer(rstd + row0, left, 4, 4), lane == 0 ? group * 4 : OUTSIDE, rs);
        if constexpr (G <= 64) load_row(tile + gridDim.x);
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
    __shared__ float lds[64];
    int turn = 0;
    const float n = (float)width;
    for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * xs;
        float t[1] = {0.f};
        for (uint64_t c = threadIdx.x * N; c < width; c += 1024 * N) {
            const Vec<T, N> v = load_vec(xr, (uint32_t)c, width);
            t[0] += pairwise<N>([&](int k) { return (float)v.e[k]; });
        }
        group_sum<1024>(t, lds, turn);
        const float mu = quotient(t[0], n, inv_width);
        float s[2] = {0.f, 0.f};
        for (uint64_t c = threadIdx.x * N; c < width; c += 1024 * N) {
            const Vec<T, N> v = load_vec(xr, (uint32_t)c, width);
            float d[N];
#pragma unroll
            for (int k = 0; k < N; ++k) d[k] = c + k < width ? (float)v.e[k] - mu : 0.f;
            s[0] += dot<N>([&](int k) { return d[k]; }, [&](int k) { return d[k]; });
            s[1] += pairwise<N>([&](int k) { return d[k]; });
        }
        group_sum<1024>(s, lds, turn);
        const Statistics st = row_statistics(s[0], s[1], inv_width, eps);
        const float rs = st.rstd, shift = -st.off * rs;
        for (uint64_t c = threadIdx.x * N; c < width; c += 1024 * N) {
            Vec<T, N> v = load_vec(xr, (uint32_t)c, width);
            float wv[N], bv[N];
            load_affine<T, false>(w, affine_fp32, (uint32_t)c, width, 1.f, wv);
            load_affine<T, false>(b, affine_fp32, (uint32_t)c, width, 0.f, bv);
#pragma unroll
            for (int k = 0; k < N; ++k) v.e[k] = (T)fmaf(fmaf((float)v.e[k] - mu, rs, shift), wv[k], bv[k]);
            store_vec(y + row * width, (uint32_t)c, width, v);
        }
        if (mean && threadIdx.x == 0) { mean[row] = mu + st.off; rstd[row] = rs; }
    }
}

// ---- backward --------------------------------------------------------------------------------------------------------------
constexpr int BWD_THREADS = 1024;

template <class W> __device__ __forceinline__ void put_column(void *p, uint32_t col, float v) { ((W *)p)[col] = (W)v; }

// sums of a share of the rows for a column: of one share alone they are the results, of several each stores a row of partial sums
// [2][width]
template <class T>
__device__ __forceinline__ void store_sum(uint32_t share, uint32_t shares, int which, uint32_t col, float v, uint32_t width, float *part,
                                          void *dw, void *db, int affine_fp32)
{
    if (shares > 1) {
        part[((uint64_t)share * 2 + which) * width + col] = v;
    } else if (void *p = which ? db : dw) {
        affine_fp32 ? put_column<float>(p, col, v) : put_column<T>(p, col, v);
    }
}

// Bound by HBM: 262144 x 64 fp32 in 34 to 36 us (6.0 TB/s, a part of it cached), 131072 x 256 bf16 in 35 us (5.8 TB/s), 8192 x 4096
// bf16 in 38 us (5.4 TB/s with the partial sums); the launch that adds those takes 4 to 5 us.  1024 threads a workgroup, one
// workgroup a CU: halves or quarters of that with as many more workgroups only made more partial sums (both directions of
// 8192 x 4096 bf16: 69.7 and 76.5 us).  The next row of each group is under way as soon as this one is in fp32 registers.  (Two
// rows ahead: 43.8 instead of 41.1 us for 262144 x 64 fp32, 44.6 instead of 41.8 us for 131072 x 256 bf16.)
template <class T, int G, int ITER, Access A>
__global__ void __launch_bounds__(BWD_THREADS)
k_ln_backward(const T *__restrict__ dy, uint64_t dys, const T *__restrict__ x, uint64_t xs, const void *__restrict__ w,
              int affine_fp32, const float *__restrict__ mean, const float *__restrict__ rstd, T *__restrict__ dx, void *dw,
              void *db, float *__restrict__ part, uint64_t rows, uint32_t width, float inv_width)
{
    constexpr int N = Vec16<T>::N, GROUPS = BWD_THREADS / G;
    // sums: the groups of a wave are added by lane moves first, so LDS holds one row of G N columns per wave or group
    constexpr int SETS = G < 64 ? BWD_THREADS / 64 : GROUPS;
    __shared__ float lds[G > 64 ? 64 : 1];
    __shared__ float sums[SETS > 1 ? SETS * G * N : 1];
    int turn = 0;
    const uint32_t lane = threadIdx.x % G, group = threadIdx.x / G;
    const uint64_t x_at = group * xs, d_at = group * dys, to_at = (uint64_t)group * width;
    // no element counts twice: what lies outside the row is zero (not asked for GLOBAL, whose widths are odd for the most part)
    const bool whole = A == TINY || (A == BUFFER && width % N == 0);
    Vec<T, N> xr[ITER], dr[ITER];
    float mu, rs;
    auto load_row = [&](uint64_t tile) {
        const uint64_t row0 = tile * GROUPS;
        const int64_t left = (int64_t)(rows - row0);
        const Rows<T, A, GROUPS> from_x(x, xs, row0, group, x_at, rows, width), from_d(dy, dys, row0, group, d_at, rows, width);
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const Place p = place<N, A>(i * G + lane, width);
            xr[i] = from_x.load(p);
            dr[i] = from_d.load(p);
        }
        if constexpr (GROUPS == 1) {
            const uint64_t r = row0 < rows ? row0 : rows - 1;
            mu = mean[r];
            rs = rstd[r];
        } else {
            mu = buffer_load<float>(rows_buffer(mean + row0, left, 4, 4), group * 4);
            rs = buffer_load<float>(rows_buffer(rstd + row0, left, 4, 4), group * 4);
        }
    };
    load_row(blockIdx.x);
    // 16 columns a lane leave no registers for the weight, it is read for each row (from the cache); 8 have them
    constexpr bool HELD = N * ITER <= 8;
    float wv[HELD ? ITER : 1][N], sw[ITER][N], sb[ITER][N];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        if constexpr (HELD) load_affine<T, A != TINY>(w, affine_fp32, place<N, A>(i * G + lane, width).at, width, 1.f, wv[i]);
#pragma unroll
        for (int k = 0; k < N; ++k) sw[i][k] = sb[i][k] = 0.f;
    }
    for (uint64_t tile = blockIdx.x; tile * GROUPS < rows; tile += gridDim.x) {
        const uint64_t row0 = tile * GROUPS, row = row0 + group;
        float h[ITER][N], g[ITER][N], t[2] = {0.f, 0.f};
        const float rs0 = rs;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            if constexpr (A == GLOBAL && GROUPS > 1) dr[i] = kept(dr[i], row < rows);  // (a row past the end came as the last one)
#pragma unroll
            for (int k = 0; k < N; ++k) {
                g[i][k] = (float)dr[i].e[k];
                h[i][k] = ((float)xr[i].e[k] - mu) * rs0;
            }
        }
        if constexpr (HELD) load_row(tile + gridDim.x);
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            if constexpr (!HELD) {
                uint32_t at = place<N, A>(i * G + lane, width).at;
                asm volatile("" : "+v"(at));  // (or the compiler takes the loads out of the loop, and spills)
                load_affine<T, A != TINY>(w, affine_fp32, at, width, 1.f, wv[0]);
            }
#pragma unroll
            for (int k = 0; k < N; ++k) {
                sw[i][k] = fmaf(g[i][k], h[i][k], sw[i][k]);
                sb[i][k] += g[i][k];
                g[i][k] *= wv[HELD ? i : 0][k];
            }
            if (A != GLOBAL && whole) {
                t[0] += pairwise<N>([&](int k) { return g[i][k]; });
                t[1] += dot<N>([&](int k) { return g[i][k]; }, [&](int k) { return h[i][k]; });
            } else {
                const int twice = (int)place<N, A>(i * G + lane, width).twice;
                float once[N];
#pragma unroll
                for (int k = 0; k < N; ++k) once[k] = k >= twice ? g[i][k] : 0.f;
                t[0] += pairwise<N>([&](int k) { return once[k]; });
                t[1] += dot<N>([&](int k) { return once[k]; }, [&](int k) { return h[i][k]; });
            }
        }
        if (dx) {  // (the same for every thread)
            group_sum<G>(t, lds, turn);
            const float a = t[0] * inv_width, c = t[1] * inv_width;
            const Rows<T, A, GROUPS> to(dx, width, row0, group, to_at, rows, width);
#pragma unroll
            for (int i = 0; i < ITER; ++i) {
                Vec<T, N> o;
#pragma unroll
                for (int k = 0; k < N; ++k) o.e[k] = (T)(rs0 * fmaf(-h[i][k], c, g[i][k] - a));
                to.store(place<N, A>(i * G + lane, width), o);
            }
        }
        if constexpr (!HELD) load_row(tile + gridDim.x);
    }
    if (!dw && !db) return;
    // the sum of element k of vector i of a lane is a column's where it counts
    auto put_sum = [&](int which, int i, uint32_t of_lane, int k, float v) {
        const Place p = place<N, A>(i * G + of_lane, width);
        if (k >= (int)p.twice && p.at + k < width)
            store_sum<T>(blockIdx.x, gridDim.x, which, p.at + k, v, width, part, dw, db, affine_fp32);
    };
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            float(&s)[N] = which ? sb[i] : sw[i];
            if constexpr (SETS == 1) {
#pragma unroll
                for (int k = 0; k < N; ++k) put_sum(which, i, lane, k, s[k]);
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
                    float v = sums[c];
                    for (int q = 1; q < SETS; ++q) v += sums[q * (G * N) + c];
                    put_sum(which, i, c % G, c / G, v);
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
                load_affine<T, false>(w, affine_fp32, (uint32_t)at, width, 1.f, wv);
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

// long rows: dw and db alone, a workgroup for 1024 N columns (blockIdx.x: the axis that takes more than 65535) of a share of the rows
// (blockIdx.y)
template <class T>
__global__ void __launch_bounds__(BWD_THREADS)
k_ln_backward_long_columns(const T *__restrict__ dy, uint64_t dys, const T *__restrict__ x, uint64_t xs,
                           const float *__restrict__ mean, const float *__restrict__ rstd, float *__restrict__ part, void *dw,
                           void *db, int affine_fp32, uint64_t rows, uint32_t width)
{
    constexpr int N = Vec16<T>::N;
    const Place p = place<N, GLOBAL>(blockIdx.x * BWD_THREADS + threadIdx.x, width);
    if (p.twice >= N) return;
    float sw[N] = {}, sb[N] = {};
    for (uint64_t row0 = blockIdx.y; row0 < rows; row0 += 4ull * gridDim.y) {  // four rows under way
        Vec<T, N> xv[4], dv[4];
        float mu[4], rs[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint64_t r = row0 + (uint64_t)u * gridDim.y, row = r < rows ? r : rows - 1;
            __builtin_memcpy(&xv[u], x + row * xs + p.at, sizeof(xv[u]));
            __builtin_memcpy(&dv[u], dy + row * dys + p.at, sizeof(dv[u]));
            mu[u] = mean[row];
            rs[u] = rstd[row];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (row0 + (uint64_t)u * gridDim.y >= rows) break;
#pragma unroll
            for (int k = 0; k < N; ++k) {
                sw[k] = fmaf((float)dv[u].e[k], ((float)xv[u].e[k] - mu[u]) * rs[u], sw[k]);
                sb[k] += (float)dv[u].e[k];
            }
        }
    }
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (k >= (int)p.twice) {
            store_sum<T>(blockIdx.y, gridDim.y, 0, p.at + k, sw[k], width, part, dw, db, affine_fp32);
            store_sum<T>(blockIdx.y, gridDim.y, 1, p.at + k, sb[k], width, part, dw, db, affine_fp32);
        }
}

// the partial sums [n][2 width] of 16 columns at a time, 64 of them at once; n = 0: no rows
constexpr uint32_t FINISH_MOST = 1u << 20;  // workgroups: a grid has less than 2^32 threads
template <class T>
__global__ void __launch_bounds__(1024)
k_ln_backward_finish(const float *__restrict__ part, uint32_t n, uint32_t width, void *dw, void *db, int affine_fp32)
{
    __shared__ float sums[16][16];
    for (uint64_t col0 = (uint64_t)blockIdx.x * 16; col0 < 2ull * width; col0 += (uint64_t)gridDim.x * 16) {
        const uint64_t col = col0 + threadIdx.x % 16;
        float acc = 0.f;
        if (col < 2ull * width)
#pragma unroll 8
            for (uint32_t s = threadIdx.x / 16; s < n; s += 64) acc += part[s * 2ull * width + col];
        acc += __shfl_xor(acc, 16, 64);
        acc += __shfl_xor(acc, 32, 64);
        if ((threadIdx.x & 63) < 16) sums[threadIdx.x >> 6][threadIdx.x & 15] = acc;
        __syncthreads();
        if (threadIdx.x < 16 && col < 2ull * width) {
            float v = sums[0][threadIdx.x];
            for (int q = 1; q < 16; ++q) v += sums[q][threadIdx.x];
            void *p = col < width ? dw : db;
            const uint32_t c = (uint32_t)(col < width ? col : col - width);
            if (p) affine_fp32 ? put_column<float>(p, c, v) : put_column<T>(p, c, v);
        }
        __syncthreads();
    }
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

// f(G, ITER) for rows of `width`: 1 vector a lane up to a wave, 8 columns a lane above it, the smallest G that covers the row.
// (16 columns a lane of half as large groups: 74 instead of 69 us for both directions of 8192 x 4096 bf16.)  The widest group
// takes more, as many as the registers hold: forward 16, backward (two sums and two inputs a column) 16 of 16 bits, 12 of fp32;
// wider rows, and in the backward pass 16-bit ones at odd addresses above 8192, go the long way.
constexpr uint32_t FORWARD_MOST = 16384;
constexpr uint32_t backward_most(uint32_t dtype) { return dtype == DT_F32 ? 12288 : 16384; }

template <class T, uint32_t MOST, class F>
int row_shape(uint32_t width, F f)
{
    constexpr uint32_t N = Vec16<T>::N;
    if (width <= 64 * N) return narrow_group<(int)N>(width, [&](auto g) { return f(g, Int<1>{}); });
    if constexpr (N < 8)
        if (width <= 64 * 8) return f(Int<64>{}, Int<8 / N>{});
    if (width <= 128 * 8) return f(Int<128>{}, Int<8 / N>{});
    if (width <= 256 * 8) return f(Int<256>{}, Int<8 / N>{});
    if (width <= 512 * 8) return f(Int<512>{}, Int<8 / N>{});
    if (width <= 1024 * 8) return f(Int<1024>{}, Int<8 / N>{});
    return f(Int<1024>{}, Int<MOST / (1024 * N)>{});
}

// BUFFER needs 4-byte addresses and `together` rows within the reach of 31-bit offsets
Access access_of(uint32_t width, uint32_t dtype, const void *a, uint64_t as, const void *b, uint64_t bs, const void *c, uint64_t cs,
                 uint32_t together)
{
    const uint64_t size = dtype_size(dtype), most = as > bs ? (as > cs ? as : cs) : (bs > cs ? bs : cs);
    if (width * size < 16) return TINY;
    return most < (1ull << 30) && most * size * together < BUFFER_MOST / 2 &&
                   (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | as * size | bs * size | cs * size) & 3) == 0
               ? BUFFER : GLOBAL;
}

// Shares of the rows in the backward pass, each with its row of partial sums.  Rows in registers: a workgroup a share, a CU a
// workgroup.  Long rows: the columns' blocks are workgroups as well, so as many shares as give two a CU, and no more than 128 rows to
// one.  (One row a share up to 256 of them took 2 GB of partial sums for 256 rows of 2^20 fp32, twice the input; now 16 MB.)
uint32_t backward_groups(uint64_t rows, uint32_t width, uint32_t dtype)
{
    if (rows == 0) return 0;
    uint64_t per = 1, most = CUS;
    if (width <= backward_most(dtype)) {
        ln_type(dtype, [&](auto t) {
            return row_shape<decltype(t), backward_most(sizeof(t) == 4 ? DT_F32 : DT_F16)>(width, [&](auto g, auto) {
                per = BWD_THREADS / decltype(g)::value;
                return 0;
            });
        });
    } else {
        const uint64_t blocks = nsr_div_up(width, BWD_THREADS * (16 / dtype_size(dtype)));
        const uint64_t few = (2 * CUS + blocks - 1) / blocks, deep = (rows + 127) / 128;
        most = deep > few ? deep : few;
        if (most > CUS) most = CUS;
    }
    const uint64_t tiles = (rows + per - 1) / per;
    // few rows: one workgroup does them all and needs no second launch (up to 4 tiles no slower alone, 12.9 instead of 16.8 us a
    // call in a row of calls; 8 tiles are slower alone)
    if (tiles <= 4) return 1;
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
    if (rows == 1) x_stride = width;  // (a single row has no stride: the kernels tell rows outside by theirs)
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
            constexpr int G = decltype(g)::value, ITER = decltype(iter)::value;
            constexpr int THREADS = G > 256 ? G : 256;
            const uint64_t tiles = (rows + THREADS / G - 1) / (THREADS / G), most = G <= 64 ? 64 * CUS : 8 * CUS * 256 / THREADS;
            const Access access = access_of(width, dtype, x, x_stride, y, width, x, x_stride, THREADS / G);
            auto kernel = access == BUFFER ? k_ln_forward<T, G, ITER, BUFFER> : k_ln_forward<T, G, ITER, GLOBAL>;
            if constexpr (G == 1)
                if (access == TINY) kernel = k_ln_forward<T, G, ITER, TINY>;
            hipLaunchKernelGGL(kernel, dim3((uint32_t)(tiles < most ? tiles : most)), dim3(THREADS), 0, (hipStream_t)stream,
                               (const T *)x, x_stride, weight, bias, fp32, (T *)y, mean, rstd, rows, width, inv, eps);
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
    if (rows == 1) x_stride = dy_stride = width;  // (a single row has no stride: the kernels tell rows outside by theirs)
    hipStream_t st = (hipStream_t)stream;
    return ln_type(dtype, [&](auto t) {
        using T = decltype(t);
        // (more than 8 columns a lane: in registers by buffer instructions only, the other form's addresses would not fit)
        const bool wide = width > 8 * BWD_THREADS && access_of(width, dtype, x, x_stride, dx, width, dy, dy_stride, 1) != BUFFER;
        if (groups && width <= backward_most(dtype) && !wide) {
            row_shape<T, backward_most(sizeof(T) == 4 ? DT_F32 : DT_F16)>(width, [&](auto g, auto iter) {
                constexpr int G = decltype(g)::value, ITER = decltype(iter)::value;
                const Access access = access_of(width, dtype, x, x_stride, dx, width, dy, dy_stride, BWD_THREADS / G);
                auto kernel = k_ln_backward<T, G, ITER, BUFFER>;
                if constexpr (Vec16<T>::N * ITER <= 8)
                    if (access == GLOBAL) kernel = k_ln_backward<T, G, ITER, GLOBAL>;
                if constexpr (G == 1)
                    if (access == TINY) kernel = k_ln_backward<T, G, ITER, TINY>;
                hipLaunchKernelGGL(kernel, dim3(groups), dim3(BWD_THREADS), 0, st,
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
                hipLaunchKernelGGL((k_ln_backward_long_columns<T>), dim3(nsr_div_up(width, BWD_THREADS * Vec16<T>::N), groups),
                                   dim3(BWD_THREADS), 0, st, (const T *)dy, dy_stride, (const T *)x, x_stride, mean, rstd,
                                   workspace, dweight, dbias, fp32, rows, width);
        }
        const uint32_t columns = (uint32_t)nsr_div_up(2ull * width, 16);
        if (affine && groups != 1)
            hipLaunchKernelGGL((k_ln_backward_finish<T>), dim3(columns < FINISH_MOST ? columns : FINISH_MOST), dim3(1024), 0, st,
                               workspace, groups, width, dweight, dbias, fp32);
        NSR_CHECK_LAUNCH("nsr_layer_norm_backward");
        return NSR_OK;
    });
}
