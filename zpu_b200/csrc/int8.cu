// The linear layer in 8-bit integers: rows quantised with one scale each,
//   scale = max |x| / 127,  q = round-half-to-even(x / scale)
// (a row of zeros keeps scale 0; a row with a NaN or an infinity gets scale
// NaN and q = 0, so only its own outputs become NaN), and the product
//   y[m, n] = (sum over k of a[m, k] * b[n, k]) * sa[m] * sb[n] + bias[n]
// whose sum is exact in 32-bit integers.
#include "head.cuh"

namespace zc {
namespace {

constexpr int NT = 256;
// 131071 * 128 * 128 < 2^31: no sum of that many products leaves 32 bits.
constexpr int64_t kMaxInner = 131071;

template <typename T>
__global__ void __launch_bounds__(NT) quantize_kernel(const T *x, int64_t ldx, int8_t *q, int64_t ldq, float *scale,
                                                      int64_t cols) {
    __shared__ float sm[NT / 32];
    const int64_t row = blockIdx.x;
    const T *xr = x + row * ldx;
    float m = 0.0f;
    for (int64_t c = threadIdx.x; c < cols; c += NT) m = max_nan(m, fabsf(to_f(xr[c])));
    m = warp_max_nan(m);
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = m;
    __syncthreads();
    m = sm[0];
    for (int w = 1; w < NT / 32; w++) m = max_nan(m, sm[w]);
    const float s = isfinite(m) ? m / 127.0f : NAN;
    for (int64_t c = threadIdx.x; c < cols; c += NT) {
        const float v = fminf(fmaxf(rintf(to_f(xr[c]) / s), -127.0f), 127.0f);
        q[row * ldq + c] = s > 0.0f ? (int8_t)(int)v : (int8_t)0;
    }
    if (threadIdx.x == 0) scale[row] = s;
}

// A 64 x 64 tile of the product per block, 64 bytes of the inner axis at a
// time through shared memory, four products an instruction.
template <typename T>
__global__ void __launch_bounds__(NT) int8_matmul_kernel(const int8_t *a, int64_t lda, const float *sa, const int8_t *b,
                                                         int64_t ldb, const float *sb, const float *bias, T *out,
                                                         int64_t ldo, int64_t m, int64_t n, int64_t k) {
    __shared__ int ta[64][17], tb[64][17];
    const int64_t m0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    for (int64_t k0 = 0; k0 < k; k0 += 64) {
        __syncthreads();
        for (int i = threadIdx.x; i < 64 * 64; i += NT) {
            const int r = i >> 6, c = i & 63;
            ((int8_t *)&ta[r][0])[c] = m0 + r < m && k0 + c < k ? a[(m0 + r) * lda + k0 + c] : (int8_t)0;
            ((int8_t *)&tb[r][0])[c] = n0 + r < n && k0 + c < k ? b[(n0 + r) * ldb + k0 + c] : (int8_t)0;
        }
        __syncthreads();
#pragma unroll
        for (int p = 0; p < 16; p++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = __dp4a(ta[ty * 4 + i][p], tb[tx + 16 * j][p], acc[i][j]);
    }
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) {
            const int64_t r = m0 + ty * 4 + i, c = n0 + tx + 16 * j;
            if (r < m && c < n) {
                const float v = (float)acc[i][j] * sa[r] * sb[c];
                out[r * ldo + c] = from_f<T>(bias ? v + bias[c] : v);
            }
        }
}

int quantize(int dtype, const void *x, int64_t ldx, int8_t *q, int64_t ldq, float *scale, int64_t rows, int64_t cols,
             cudaStream_t s) {
    if (rows == 0) return ZPUCUDA_OK;
    ZC_HEAD_TYPE(dtype, T, quantize_kernel<T><<<(unsigned)rows, NT, 0, s>>>((const T *)x, ldx, q, ldq, scale, cols));
    ZC_LAUNCHED("quantize_kernel");
    return ZPUCUDA_OK;
}

int product(const int8_t *a, int64_t lda, const float *sa, const int8_t *b, int64_t ldb, const float *sb,
            const float *bias, int dtype, void *out, int64_t ldo, int64_t m, int64_t n, int64_t k, cudaStream_t s) {
    if (m == 0 || n == 0) return ZPUCUDA_OK;
    dim3 grid((unsigned)((n + 63) / 64), (unsigned)((m + 63) / 64));
    ZC_HEAD_TYPE(dtype, T,
                 int8_matmul_kernel<T><<<grid, NT, 0, s>>>(a, lda, sa, b, ldb, sb, bias, (T *)out, ldo, m, n, k));
    ZC_LAUNCHED("int8_matmul_kernel");
    return ZPUCUDA_OK;
}

int check_product(const char *who, const float *sb, const int8_t *b, int64_t ldb, const float *bias, int dtype,
                  const void *out, int64_t ldo, int64_t m, int64_t n, int64_t k) {
    if (m < 0 || n < 0 || k < 0) return head_error(ZPUCUDA_ERR_INVALID_SHAPE, who, "a size is negative");
    if (k > kMaxInner) return head_error(ZPUCUDA_ERR_NOT_SUPPORTED, who, "an inner size above 131071 could leave 32 bits");
    if (m > 64 * 65535ll || n > 0x7fffffff - 255) return head_error(ZPUCUDA_ERR_NOT_SUPPORTED, who, "more than 4194240 rows or 2^31 - 256 columns");
    ZC_TRY(check_matrix(who, "out", out, dtype, ldo, m, n));
    if (ldb < k) return head_error(ZPUCUDA_ERR_INVALID_SHAPE, who, "b: row pitch below the row's length");
    if (n > 0 && ((k > 0 && !b) || !sb)) return head_error(ZPUCUDA_ERR_INVALID_ARGUMENT, who, "b or its scales: null pointer");
    (void)bias;
    return ZPUCUDA_OK;
}

}  // namespace
}  // namespace zc

using namespace zc;

extern "C" {

int zpucuda_int8_quantize(int dtype, const void *d_x, int64_t ldx, int8_t *d_q, int64_t ldq, float *d_scale,
                          int64_t rows, int64_t cols, void *stream) {
    if (rows < 0 || cols < 0) return set_error(ZPUCUDA_ERR_INVALID_SHAPE, "int8_quantize: a size is negative");
    if (rows > 0x7fffffff) return set_error(ZPUCUDA_ERR_NOT_SUPPORTED, "int8_quantize: more than 2^31 - 1 rows");
    ZC_TRY(check_matrix("int8_quantize", "x", d_x, dtype, ldx, rows, cols));
    if (ldq < cols) return set_error(ZPUCUDA_ERR_INVALID_SHAPE, "int8_quantize: q: row pitch below the row's length");
    if (rows > 0 && ((cols > 0 && !d_q) || !d_scale))
        return set_error(ZPUCUDA_ERR_INVALID_ARGUMENT, "int8_quantize: q or scale: null pointer");
    return quantize(dtype, d_x, ldx, d_q, ldq, d_scale, rows, cols, resolve_stream(stream));
}

int zpucuda_int8_matmul(const int8_t *d_a, int64_t lda, const float *d_sa, const int8_t *d_b, int64_t ldb,
                        const float *d_sb, const float *d_bias, int dtype, void *d_out, int64_t ldo, int64_t m,
                        int64_t n, int64_t k, void *stream) {
    ZC_TRY(check_product("int8_matmul", d_sb, d_b, ldb, d_bias, dtype, d_out, ldo, m, n, k));
    if (lda < k) return set_error(ZPUCUDA_ERR_INVALID_SHAPE, "int8_matmul: a: row pitch below the row's length");
    if (m > 0 && ((k > 0 && !d_a) || !d_sa))
        return set_error(ZPUCUDA_ERR_INVALID_ARGUMENT, "int8_matmul: a or its scales: null pointer");
    return product(d_a, lda, d_sa, d_b, ldb, d_sb, d_bias, dtype, d_out, ldo, m, n, k, resolve_stream(stream));
}

int zpucuda_int8_linear(int dtype, const void *d_x, int64_t ldx, const int8_t *d_w, int64_t ldw, const float *d_sw,
                        const float *d_bias, void *d_y, int64_t ldy, int64_t rows, int64_t cols, int64_t inner,
                        void *d_work, int64_t work_bytes, void *stream) {
    ZC_TRY(check_product("int8_linear", d_sw, d_w, ldw, d_bias, dtype, d_y, ldy, rows, cols, inner));
    ZC_TRY(check_matrix("int8_linear", "x", d_x, dtype, ldx, rows, inner));
    if (rows == 0 || cols == 0) return ZPUCUDA_OK;
    if (!d_work || work_bytes < zpucuda_int8_linear_work(rows, inner) || !aligned_to(d_work, 16))
        return set_error(ZPUCUDA_ERR_INVALID_ARGUMENT, "int8_linear: work: null, too small or not 16-byte aligned");
    cudaStream_t s = resolve_stream(stream);
    const int64_t ldq = (inner + 15) / 16 * 16;
    int8_t *q = (int8_t *)d_work;
    float *scale = (float *)(q + rows * ldq);
    ZC_TRY(quantize(dtype, d_x, ldx, q, ldq, scale, rows, inner, s));
    return product(q, ldq, scale, d_w, ldw, d_sw, d_bias, dtype, d_y, ldy, rows, cols, inner, s);
}

int64_t zpucuda_int8_linear_work(int64_t rows, int64_t inner) {
    if (rows < 0 || inner < 0) return 0;
    return rows * ((inner + 15) / 16 * 16) + rows * 4;
}

}  // extern "C"
