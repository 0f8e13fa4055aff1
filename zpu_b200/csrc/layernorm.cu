// Layer norm over the last axis, forward and backward (nn.layerNorm,
// restated for a batch of rows):
//   mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps)
//   y = (x - mu) * rstd * gamma + beta
// and with xhat = (x - mu) * rstd, g = dy * gamma:
//   dx = rstd * (g - mean(g) - xhat * mean(g * xhat))
//   dgamma = sum over rows of dy * xhat,  dbeta = sum over rows of dy.
#include "head.cuh"

namespace zc {
namespace {

constexpr int NT = 256;

// Sums of two values over the block; every thread gets both.
__device__ __forceinline__ float2 block_sum2(float a, float b, float2 *sm) {
    a = warp_sum(a);
    b = warp_sum(b);
    __syncthreads();  // the previous sum's readers are done
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    float2 t = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < NT / 32; w++) {
        t.x += sm[w].x;
        t.y += sm[w].y;
    }
    return t;
}

template <typename T>
__global__ void __launch_bounds__(NT) ln_kernel(const T *x, int64_t ldx, int wt, const void *gamma, const void *beta,
                                                T *y, int64_t ldy, float *mean, float *rstd, int64_t cols, float eps) {
    __shared__ float2 sm[NT / 32];
    const int64_t row = blockIdx.x;
    const T *xr = x + row * ldx;
    T *yr = y + row * ldy;
    float s = 0.0f;
    for (int64_t c = threadIdx.x; c < cols; c += NT) s += to_f(xr[c]);
    const float mu = block_sum2(s, 0.0f, sm).x / (float)cols;
    // The mean of what the rounded mean leaves is taken off again: rows far
    // from zero keep the digits that a 32-bit mean alone would cost them.
    float e = 0.0f, v = 0.0f;
    for (int64_t c = threadIdx.x; c < cols; c += NT) {
        const float d = to_f(xr[c]) - mu;
        e += d;
        v += d * d;
    }
    const float2 t = block_sum2(e, v, sm);
    const float rest = t.x / (float)cols;
    float var = t.y / (float)cols - rest * rest;
    var = var < 0.0f ? 0.0f : var;  // NaN stays
    const float rs = 1.0f / sqrtf(var + eps);
    for (int64_t c = threadIdx.x; c < cols; c += NT) {
        const float g = gamma ? load_f(gamma, wt, c) : 1.0f, b = beta ? load_f(beta, wt, c) : 0.0f;
        yr[c] = from_f<T>(((to_f(xr[c]) - mu) - rest) * rs * g + b);
    }
    if (threadIdx.x == 0) {
        if (mean) mean[row] = mu + rest;
        if (rstd) rstd[row] = rs;
    }
}

template <typename T>
__global__ void __launch_bounds__(NT) ln_dx_kernel(const T *dy, int64_t lddy, const T *x, int64_t ldx,
                                                   const float *mean, const float *rstd, int wt, const void *gamma,
                                                   T *dx, int64_t lddx, int64_t cols) {
    __shared__ float2 sm[NT / 32];
    const int64_t row = blockIdx.x;
    const T *xr = x + row * ldx, *dr = dy + row * lddy;
    T *o = dx + row * lddx;
    const float mu = mean[row], rs = rstd[row];
    float a = 0.0f, b = 0.0f;
    for (int64_t c = threadIdx.x; c < cols; c += NT) {
        const float g = to_f(dr[c]) * (gamma ? load_f(gamma, wt, c) : 1.0f);
        a += g;
        b += g * ((to_f(xr[c]) - mu) * rs);
    }
    const float2 t = block_sum2(a, b, sm);
    const float ma = t.x / (float)cols, mb = t.y / (float)cols;
    for (int64_t c = threadIdx.x; c < cols; c += NT) {
        const float g = to_f(dr[c]) * (gamma ? load_f(gamma, wt, c) : 1.0f);
        o[c] = from_f<T>(rs * (g - ma - (to_f(xr[c]) - mu) * rs * mb));
    }
}

// One block sums 32 columns over all rows, eight rows at a time.
template <typename T>
__global__ void __launch_bounds__(NT) ln_dw_kernel(const T *dy, int64_t lddy, const T *x, int64_t ldx,
                                                   const float *mean, const float *rstd, int wt, void *dgamma,
                                                   void *dbeta, int64_t rows, int64_t cols) {
    __shared__ float sg[8][33], sb[8][33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    float g = 0.0f, b = 0.0f;
    if (c < cols)
        for (int64_t r = w; r < rows; r += 8) {
            const float d = to_f(dy[r * lddy + c]);
            b += d;
            g += d * ((to_f(x[r * ldx + c]) - mean[r]) * rstd[r]);
        }
    sg[w][lane] = g;
    sb[w][lane] = b;
    __syncthreads();
    if (w == 0 && c < cols) {
        for (int i = 1; i < 8; i++) {
            g += sg[i][lane];
            b += sb[i][lane];
        }
        if (dgamma) store_f(dgamma, wt, c, g);
        if (dbeta) store_f(dbeta, wt, c, b);
    }
}

}  // namespace
}  // namespace zc

using namespace zc;

extern "C" {

int zpucuda_layer_norm(int dtype, const void *d_x, int64_t ldx, int wtype, const void *d_gamma, const void *d_beta,
                       void *d_y, int64_t ldy, float *d_mean, float *d_rstd, int64_t rows, int64_t cols, double eps,
                       void *stream) {
    if (rows < 0 || cols < 1) return set_error(ZPUCUDA_ERR_INVALID_SHAPE, "layer_norm: rows >= 0 and cols >= 1 are wanted");
    if (!(eps >= 0.0)) return set_error(ZPUCUDA_ERR_INVALID_ARGUMENT, "layer_norm: eps is negative or NaN");
    ZC_TRY(check_matrix("layer_norm", "x", d_x, dtype, ldx, rows, cols));
    ZC_TRY(check_matrix("layer_norm", "y", d_y, dtype, ldy, rows, cols));
    if (d_gamma) ZC_TRY(check_matrix("layer_norm", "gamma", d_gamma, wtype, cols, 1, cols));
    if (d_beta) ZC_TRY(check_matrix("layer_norm", "beta", d_beta, wtype, cols, 1, cols));
    if (rows == 0) return ZPUCUDA_OK;
    cudaStream_t s = resolve_stream(stream);
    ZC_HEAD_TYPE(dtype, T,
                 ln_kernel<T><<<(unsigned)rows, NT, 0, s>>>((const T *)d_x, ldx, wtype, d_gamma, d_beta, (T *)d_y, ldy,
                                                            d_mean, d_rstd, cols, (float)eps));
    ZC_LAUNCHED("ln_kernel");
    return ZPUCUDA_OK;
}

int zpucuda_layer_norm_grad(int dtype, const void *d_dy, int64_t lddy, const void *d_x, int64_t ldx,
                            const float *d_mean, const float *d_rstd, int wtype, const void *d_gamma, void *d_dx,
                            int64_t lddx, void *d_dgamma, void *d_dbeta, int64_t rows, int64_t cols, void *stream) {
    if (rows < 0 || cols < 1)
        return set_error(ZPUCUDA_ERR_INVALID_SHAPE, "layer_norm_grad: rows >= 0 and cols >= 1 are wanted");
    ZC_TRY(check_matrix("layer_norm_grad", "dy", d_dy, dtype, lddy, rows, cols));
    ZC_TRY(check_matrix("layer_norm_grad", "x", d_x, dtype, ldx, rows, cols));
    if (d_dx) ZC_TRY(check_matrix("layer_norm_grad", "dx", d_dx, dtype, lddx, rows, cols));
    if (d_gamma) ZC_TRY(check_matrix("layer_norm_grad", "gamma", d_gamma, wtype, cols, 1, cols));
    if (d_dgamma) ZC_TRY(check_matrix("layer_norm_grad", "dgamma", d_dgamma, wtype, cols, 1, cols));
    if (d_dbeta) ZC_TRY(check_matrix("layer_norm_grad", "dbeta", d_dbeta, wtype, cols, 1, cols));
    if (rows > 0 && (!d_mean || !d_rstd))
        return set_error(ZPUCUDA_ERR_INVALID_ARGUMENT, "layer_norm_grad: mean or rstd is null");
    cudaStream_t s = resolve_stream(stream);
    if (d_dgamma || d_dbeta) {
        ZC_HEAD_TYPE(dtype, T,
                     ln_dw_kernel<T><<<(unsigned)((cols + 31) / 32), NT, 0, s>>>((const T *)d_dy, lddy, (const T *)d_x,
                                                                                ldx, d_mean, d_rstd, wtype, d_dgamma,
                                                                                d_dbeta, rows, cols));
        ZC_LAUNCHED("ln_dw_kernel");
    }
    if (d_dx && rows > 0) {
        ZC_HEAD_TYPE(dtype, T,
                     ln_dx_kernel<T><<<(unsigned)rows, NT, 0, s>>>((const T *)d_dy, lddy, (const T *)d_x, ldx, d_mean,
                                                                   d_rstd, wtype, d_gamma, (T *)d_dx, lddx, cols));
        ZC_LAUNCHED("ln_dx_kernel");
    }
    return ZPUCUDA_OK;
}

}  // extern "C"
