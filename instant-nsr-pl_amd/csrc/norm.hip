// Layer norm over the last axis, forward and backward, with the reduction of the weight's and the bias' gradients.
//   mu = mean(x), s = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) s, y = h w + b
//   dx = s (g - mean(g) - h mean(g h)) with g = dy w,  dw = sum over rows of dy h,  db = sum over rows of dy
// Statistics, sums and products in fp32 whatever the storage type; the variance from centred values (x is read again or held).
#include "elem.h"

namespace {

constexpr int LN_THREADS = 256;
constexpr uint32_t LN_SPLITS = 256;

template <class T, class W>
__global__ void __launch_bounds__(LN_THREADS)
k_ln_forward(const T *__restrict__ x, uint64_t xs, const W *__restrict__ w, const W *__restrict__ b, T *__restrict__ y,
             float *__restrict__ mean, float *__restrict__ rstd, uint64_t rows, uint32_t width, float inv_width, float eps)
{
    const uint32_t lane = threadIdx.x & 63;
    for (uint64_t row = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (uint64_t)gridDim.x * 4) {
        const T *xr = x + row * xs;
        float s = 0.f, q = 0.f;
        for (uint32_t i = lane; i < width; i += 64) s += (float)xr[i];
        const float mu = wave_sum(s) * inv_width;
        for (uint32_t i = lane; i < width; i += 64) { const float c = (float)xr[i] - mu; q += c * c; }
        const float rs = 1.f / sqrtf(wave_sum(q) * inv_width + eps);
        for (uint32_t i = lane; i < width; i += 64) {
            float v = ((float)xr[i] - mu) * rs;
            if (w) v *= (float)w[i];
            if (b) v += (float)b[i];
            y[row * width + i] = (T)v;
        }
        if (lane == 0 && mean) { mean[row] = mu; rstd[row] = rs; }
    }
}

template <class T, class W>
__global__ void __launch_bounds__(LN_THREADS)
k_ln_backward_rows(const T *__restrict__ dy, uint64_t dys, const T *__restrict__ x, uint64_t xs, const W *__restrict__ w,
                   const float *__restrict__ mean, const float *__restrict__ rstd, T *__restrict__ dx, uint64_t rows,
                   uint32_t width, float inv_width)
{
    const uint32_t lane = threadIdx.x & 63;
    for (uint64_t row = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (uint64_t)gridDim.x * 4) {
        const T *xr = x + row * xs, *dr = dy + row * dys;
        const float mu = mean[row], rs = rstd[row];
        float a = 0.f, c = 0.f;
        for (uint32_t i = lane; i < width; i += 64) {
            const float g = (float)dr[i] * (w ? (float)w[i] : 1.f);
            a += g;
            c += g * (((float)xr[i] - mu) * rs);
        }
        a = wave_sum(a) * inv_width;
        c = wave_sum(c) * inv_width;
        for (uint32_t i = lane; i < width; i += 64) {
            const float g = (float)dr[i] * (w ? (float)w[i] : 1.f);
            dx[row * width + i] = (T)(rs * (g - a - ((float)xr[i] - mu) * rs * c));
        }
    }
}

// partial sums of one split of the rows for 64 columns: [split][dw | db][width]
template <class T>
__global__ void __launch_bounds__(LN_THREADS)
k_ln_backward_columns(const T *__restrict__ dy, uint64_t dys, const T *__restrict__ x, uint64_t xs,
                      const float *__restrict__ mean, const float *__restrict__ rstd, float *__restrict__ part, uint64_t rows,
                      uint32_t width)
{
    const uint32_t col = blockIdx.x * 64 + (threadIdx.x & 63), wave = threadIdx.x >> 6;
    float dw = 0.f, db = 0.f;
    if (col < width)
        for (uint64_t row = (uint64_t)blockIdx.y * 4 + wave; row < rows; row += (uint64_t)gridDim.y * 4) {
            const float d = (float)dy[row * dys + col];
            dw += d * (((float)x[row * xs + col] - mean[row]) * rstd[row]);
            db += d;
        }
    __shared__ float sh[2][LN_THREADS];
    sh[0][threadIdx.x] = dw;
    sh[1][threadIdx.x] = db;
    __syncthreads();
    if (wave == 0 && col < width)
        for (int k = 0; k < 2; ++k)
            part[((uint64_t)blockIdx.y * 2 + k) * width + col] =
                (sh[k][threadIdx.x] + sh[k][threadIdx.x + 64]) + (sh[k][threadIdx.x + 128] + sh[k][threadIdx.x + 192]);
}

template <class W>
__global__ void __launch_bounds__(LN_THREADS)
k_ln_backward_finish(const float *__restrict__ part, uint32_t splits, uint32_t width, W *__restrict__ dw, W *__restrict__ db)
{
    const uint32_t col = blockIdx.x * LN_THREADS + threadIdx.x;
    if (col >= width) return;
    float a = 0.f, c = 0.f;
    for (uint32_t s = 0; s < splits; ++s) {
        a += part[(uint64_t)s * 2 * width + col];
        c += part[((uint64_t)s * 2 + 1) * width + col];
    }
    if (dw) dw[col] = (W)a;
    if (db) db[col] = (W)c;
}

uint32_t ln_splits(uint64_t rows) { return rows < 4ull * LN_SPLITS ? nsr_div_up(rows, 4) : LN_SPLITS; }

uint32_t row_grid(uint64_t rows) { return rows < 4ull << 20 ? nsr_div_up(rows, 4) : 1u << 20; }

// calls f with a value of the storage type and one of the affine parameters' type
template <class F>
int ln_types(uint32_t dtype, uint32_t affine, F f)
{
    if (dtype == DT_F32) return f(float{}, float{});
    if (dtype == DT_F16) return affine == DT_F32 ? f(_Float16{}, float{}) : f(_Float16{}, _Float16{});
    return affine == DT_F32 ? f(__bf16{}, float{}) : f(__bf16{}, __bf16{});
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
                    !misaligned(bias, affine_dtype), "nsr_layer_norm_forward: misaligned pointer");
    return ln_types(dtype, affine_dtype, [&](auto t, auto w) {
        using T = decltype(t);
        using W = decltype(w);
        hipLaunchKernelGGL((k_ln_forward<T, W>), dim3(row_grid(rows)), dim3(LN_THREADS), 0, (hipStream_t)stream, (const T *)x,
                           x_stride, (const W *)weight, (const W *)bias, (T *)y, mean, rstd, rows, width, 1.f / (float)width,
                           eps);
        NSR_CHECK_LAUNCH("nsr_layer_norm_forward");
        return NSR_OK;
    });
}

extern "C" uint64_t nsr_layer_norm_backward_workspace_floats(uint64_t rows, uint32_t width)
{
    return (uint64_t)ln_splits(rows) * 2 * width;
}

extern "C" int nsr_layer_norm_backward(const void *dy, uint64_t dy_stride, const void *x, uint64_t x_stride, const void *weight,
                                       const float *mean, const float *rstd, void *dx, void *dweight, void *dbias,
                                       float *workspace, uint64_t rows, uint32_t width, uint32_t dtype, uint32_t affine_dtype,
                                       void *stream)
{
    const int rc = ln_check("nsr_layer_norm_backward", rows, width, dtype, affine_dtype);
    if (rc != NSR_OK) return rc;
    const bool affine = dweight || dbias;
    NSR_REQUIRE(rows == 0 || (dy && x && mean && rstd), "nsr_layer_norm_backward: NULL pointer");
    NSR_REQUIRE(rows == 0 || !affine || workspace, "nsr_layer_norm_backward: the affine gradients need the workspace");
    NSR_REQUIRE((x_stride >= width && dy_stride >= width) || rows <= 1, "nsr_layer_norm_backward: rows overlap");
    NSR_REQUIRE(!misaligned(dy, dtype) && !misaligned(x, dtype) && !misaligned(dx, dtype) && !misaligned(weight, affine_dtype) &&
                    !misaligned(dweight, affine_dtype) && !misaligned(dbias, affine_dtype) && ((uintptr_t)workspace & 3) == 0,
                "nsr_layer_norm_backward: misaligned pointer");
    const uint32_t splits = ln_splits(rows);
    return ln_types(dtype, affine_dtype, [&](auto t, auto w) {
        using T = decltype(t);
        using W = decltype(w);
        hipStream_t st = (hipStream_t)stream;
        if (dx && rows)
            hipLaunchKernelGGL((k_ln_backward_rows<T, W>), dim3(row_grid(rows)), dim3(LN_THREADS), 0, st, (const T *)dy,
                               dy_stride, (const T *)x, x_stride, (const W *)weight, mean, rstd, (T *)dx, rows, width,
                               1.f / (float)width);
        if (affine) {
            if (rows)
                hipLaunchKernelGGL((k_ln_backward_columns<T>), dim3(nsr_div_up(width, 64), splits), dim3(LN_THREADS), 0, st,
                                   (const T *)dy, dy_stride, (const T *)x, x_stride, mean, rstd, workspace, rows, width);
            hipLaunchKernelGGL((k_ln_backward_finish<W>), dim3(nsr_div_up(width, LN_THREADS)), dim3(LN_THREADS), 0, st,
                               workspace, splits, width, (W *)dweight, (W *)dbias);
        }
        NSR_CHECK_LAUNCH("nsr_layer_norm_backward");
        return NSR_OK;
    });
}
