// Layer norm over the last axis, forward and backward (nn.layerNorm,
// restated for a batch of rows):
//   mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps)
//   y = (x - mu) * rstd * gamma + beta
// and with xhat = (x - mu) * rstd, g = dy * gamma:
//   dx = rstd * (g - mean(g) - xhat * mean(g * xhat))
//   dgamma = sum over rows of dy * xhat,  dbeta = sum over rows of dy.
// HBM bounds both: a row is read once into registers, reduced there, and
// written.  The gradient's blocks walk rows and keep their columns' sums of
// dgamma and dbeta in registers; one row of sums a block goes to the caller's
// workspace, and a second kernel adds those up in the blocks' order, so a
// result does not depend on the run.
#include "head.cuh"

namespace zc {
namespace {

constexpr int NT = 256;
constexpr int kPerThread = 16;  // columns that a thread of the one-pass gradient holds
constexpr int kMaxParts = 2;    // blocks an SM of the gradient

// The weights of piece i of a row (N from column i * N on, `have` of them), as
// f32; `dflt` without any.
template <int N>
__device__ __forceinline__ void load_w(const void *p, int wt, int64_t i, int have, float dflt, float (&f)[N]) {
    const int64_t c = i * N;
    if (p && have == N && ((uintptr_t)p & 15) == 0) {
        if (wt == ZPUCUDA_F32) {
#pragma unroll
            for (int e = 0; e < N; e += 4) {
                const float4 v = *(const float4 *)((const float *)p + c + e);
                f[e] = v.x;
                f[e + 1] = v.y;
                f[e + 2] = v.z;
                f[e + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < N; e += 4) {
                const uint2 v = *(const uint2 *)((const uint16_t *)p + c + e);
                const uint32_t h[4] = {v.x & 0xffff, v.x >> 16, v.y & 0xffff, v.y >> 16};
#pragma unroll
                for (int k = 0; k < 4; k++)
                    f[e + k] = wt == ZPUCUDA_F16 ? __half2float(__ushort_as_half((unsigned short)h[k])) : __uint_as_float(h[k] << 16);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) f[e] = p && e < have ? load_f(p, wt, c + e) : dflt;
    }
}

// How many elements of piece i are in a row of cols.
template <int N>
__device__ __forceinline__ int in_row(int64_t i, int64_t cols) {
    const int64_t rest = cols - i * N;
    return rest >= N ? N : rest > 0 ? (int)rest : 0;
}

// Sums of two values over the TPR threads of a row; every thread gets both.
// sm: TPR / 32 entries of the row's own; barrier `bar` is the row's own.
template <int TPR>
__device__ __forceinline__ float2 row_sum2(float a, float b, float2 *sm, int bar) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (TPR == 32) return make_float2(a, b);
    if ((threadIdx.x & 31) == 0) sm[(threadIdx.x % TPR) >> 5] = make_float2(a, b);
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(TPR) : "memory");
    float2 t = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < TPR / 32; w++) {
        t.x += sm[w].x;
        t.y += sm[w].y;
    }
    return t;
}

// ------------------------------------------------------------------ forward

// TPR threads a row, NV pieces a thread.  NV = 0: rows too long for registers,
// read three times (from L2 after the first).
template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(TPR < NT ? NT : TPR)
    ln_kernel(const T *x, int64_t ldx, int wt, const void *gamma, const void *beta, T *y, int64_t ldy, float *mean,
              float *rstd, int64_t rows, int64_t cols, float eps) {
    constexpr int BLOCK = TPR < NT ? NT : TPR, N = kPiece<T>;
    __shared__ float2 sm[2][BLOCK / 32];
    const int64_t row = (int64_t)blockIdx.x * (BLOCK / TPR) + threadIdx.x / TPR;
    if (row >= rows) return;  // a whole warp; with TPR > 32 a block has one row
    const int t = threadIdx.x % TPR;
    const T *xr = x + row * ldx;
    T *yr = y + row * ldy;
    const int64_t n = (cols + N - 1) / N;
    const float inv = 1.0f / (float)cols;
    uint4 v[NV ? NV : 1];
    if constexpr (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; j++)
            v[j] = t + j * TPR < n ? load_piece(xr, t + j * TPR, cols) : make_uint4(0, 0, 0, 0);
    }
    // a thread's part of the three passes, over its pieces
    float s = 0.0f, d1 = 0.0f, d2 = 0.0f, mu, rest, rs;
    auto sum = [&](const uint4 &in) {  // what is past the row's end is 0
        float a[N];
        unpack<T>(in, a);
#pragma unroll
        for (int e = 0; e < N; e++) s += a[e];
    };
    auto spread = [&](const uint4 &in, int64_t i) {
        float a[N];
        unpack<T>(in, a);
        const int have = in_row<N>(i, cols);
#pragma unroll
        for (int e = 0; e < N; e++) {
            const float d = e < have ? a[e] - mu : 0.0f;
            d1 += d;
            d2 += d * d;
        }
    };
    auto put = [&](const uint4 &in, int64_t i) {  // a whole warp's pieces
        float a[N], g[N], b[N];
        unpack<T>(in, a);
        const int have = in_row<N>(i, cols);
        load_w<N>(gamma, wt, i, have, 1.0f, g);
        load_w<N>(beta, wt, i, have, 0.0f, b);
#pragma unroll
        for (int e = 0; e < N; e++) a[e] = ((a[e] - mu) - rest) * rs * g[e] + b[e];
        __syncwarp();
        store_piece(yr, i, cols, pack<T>(a));
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; j++) sum(v[j]);
    } else {
        for (int64_t i = t; i < n; i += TPR) sum(load_piece(xr, i, cols));
    }
    mu = row_sum2<TPR>(s, 0.0f, sm[0], 0).x * inv;
    // The mean of what the rounded mean leaves is taken off again: rows far
    // from zero keep the digits that a 32-bit mean alone would cost them.
    if constexpr (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; j++) spread(v[j], t + j * TPR);
    } else {
        for (int64_t i = t; i < n; i += TPR) spread(load_piece(xr, i, cols), i);
    }
    const float2 q = row_sum2<TPR>(d1, d2, sm[1], 0);
    rest = q.x * inv;
    float var = q.y * inv - rest * rest;
    var = var < 0.0f ? 0.0f : var;  // NaN stays
    rs = 1.0f / sqrtf(var + eps);
    if constexpr (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; j++) put(v[j], t + j * TPR);
    } else {
        for (int64_t i = t; i - (t & 31) < n; i += TPR) put(i < n ? load_piece(xr, i, cols) : make_uint4(0, 0, 0, 0), i);
    }
    if (t == 0) {
        if (mean) mean[row] = mu + rest;
        if (rstd) rstd[row] = rs;
    }
}

template <typename T>
int launch_ln(const T *x, int64_t ldx, int wt, const void *gamma, const void *beta, T *y, int64_t ldy, float *mean,
              float *rstd, int64_t rows, int64_t cols, float eps, cudaStream_t s) {
    const int64_t n = (cols + kPiece<T> - 1) / kPiece<T>;
    const unsigned few = (unsigned)((rows + NT / 32 - 1) / (NT / 32)), all = (unsigned)rows;
#define LN(TPR, NV)                                                                                         \
    ln_kernel<T, TPR, NV><<<TPR == 32 ? few : all, TPR < NT ? NT : TPR, 0, s>>>(x, ldx, wt, gamma, beta, y, \
                                                                               ldy, mean, rstd, rows, cols, eps)
    // a warp holds 128 pieces, 256 threads 1024, 1024 threads 4096
    if (n <= 32) LN(32, 1);
    else if (n <= 64) LN(32, 2);
    else if (n <= 128) LN(32, 4);
    else if (n <= 256) LN(256, 1);
    else if (n <= 512) LN(256, 2);
    else if (n <= 1024) LN(256, 4);
    else if (n <= 2048) LN(1024, 2);
    else if (n <= 4096) LN(1024, 4);
    else LN(1024, 0);
#undef LN
    ZC_LAUNCHED("ln_kernel");
    return ZPUCUDA_OK;
}

// ----------------------------------------------------------------- backward

// One pass: TPR threads a row, BLOCK / TPR rows of a block at a time, NV pieces a
// thread.  The next row's loads are in flight while this one is reduced and
// written.  parts: [gridDim.x][2][cols] sums, or null.  1024 threads (64
// registers each) keep the sums in shared memory, every thread its own.
template <typename T, int TPR, int NV, int BLOCK>
__global__ void __launch_bounds__(BLOCK)
    ln_grad_kernel(const T *dy, int64_t lddy, const T *x, int64_t ldx, const float *mean, const float *rstd, int wt,
                   const void *gamma, T *dx, int64_t lddx, float *parts, int64_t rows, int64_t cols) {
    constexpr int GROUPS = BLOCK / TPR, N = kPiece<T>;
    constexpr bool SHARED = BLOCK == 1024;
    __shared__ float2 sm[2][BLOCK / 32];
    extern __shared__ __align__(16) float comb[];  // [2][pitch], to add up the groups, or SHARED
    const int t = threadIdx.x % TPR, group = threadIdx.x / TPR, bar = 1 + (TPR > 32 ? group : 0);
    const int64_t n = (cols + N - 1) / N, pitch = n * N;
    const float inv = 1.0f / (float)cols;
    constexpr int K = SHARED ? 1 : NV;
    float gs[K][N], ag[K][N] = {}, ab[K][N] = {};
    auto weights = [&](int j, float (&w)[N]) { load_w<N>(gamma, wt, t + j * TPR, in_row<N>(t + j * TPR, cols), 1.0f, w); };
    if constexpr (SHARED) {
        for (int64_t c = threadIdx.x; c < 2 * pitch; c += BLOCK) comb[c] = 0.0f;
        __syncthreads();
    } else {
#pragma unroll
        for (int j = 0; j < NV; j++) weights(j, gs[j]);
    }
    uint4 vx[NV], vd[NV], px[NV], pd[NV];
    float mu = 0.0f, rs = 0.0f, pmu = 0.0f, prs = 0.0f;
    auto load = [&](int64_t row) {
        if (row >= rows) return;
        pmu = mean[row];
        prs = rstd[row];
#pragma unroll
        for (int j = 0; j < NV; j++)
            if (t + j * TPR < n) {
                px[j] = load_piece(x + row * ldx, t + j * TPR, cols);
                pd[j] = load_piece(dy + row * lddy, t + j * TPR, cols);
            }
    };
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    int64_t row = (int64_t)blockIdx.x * GROUPS + group;
    load(row);
    for (int odd = 0; row < rows; row += step, odd ^= 1) {
        mu = pmu;
        rs = prs;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            vx[j] = px[j];
            vd[j] = pd[j];
        }
        load(row + step);
        float a = 0.0f, b = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++) {  // past the row's end dy is 0, and all that follows from it
            if (t + j * TPR >= n) continue;
            float fx[N], fd[N], w[N];
            unpack<T>(vx[j], fx);
            unpack<T>(vd[j], fd);
            if constexpr (SHARED) weights(j, w);
            float *sg = comb + (t + j * TPR) * N, *sb = sg + pitch;
#pragma unroll
            for (int e = 0; e < N; e++) {
                const float xh = (fx[e] - mu) * rs, d = fd[e];
                const float gd = d * (SHARED ? w[e] : gs[SHARED ? 0 : j][e]);
                a += gd;
                b += gd * xh;
                if constexpr (SHARED) {
                    sg[e] += d * xh;
                    sb[e] += d;
                } else {
                    ag[j][e] += d * xh;
                    ab[j][e] += d;
                }
            }
        }
        if (!dx) continue;
        // two buffers: a thread that is a row ahead does not overwrite what another still reads
        const float2 q = row_sum2<TPR>(a, b, sm[odd] + group * (TPR / 32), bar);
        const float ma = q.x * inv, mb = q.y * inv;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            float fx[N], fd[N], w[N];
            unpack<T>(vx[j], fx);
            unpack<T>(vd[j], fd);
            if constexpr (SHARED) weights(j, w);
#pragma unroll
            for (int e = 0; e < N; e++) {
                const float xh = (fx[e] - mu) * rs;
                fx[e] = rs * (fd[e] * (SHARED ? w[e] : gs[SHARED ? 0 : j][e]) - ma - xh * mb);
            }
            __syncwarp();
            store_piece(dx + row * lddx, t + j * TPR, cols, pack<T>(fx));
        }
    }
    if (!parts) return;
    float *out = parts + (int64_t)blockIdx.x * 2 * cols;
    if constexpr (!SHARED) {  // the groups add up in their order
        for (int k = 0; k < GROUPS; k++) {
            __syncthreads();
            if (group == k)
#pragma unroll
                for (int j = 0; j < NV; j++) {
                    if (t + j * TPR >= n) continue;
                    float *sg = comb + (t + j * TPR) * N, *sb = sg + pitch;
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        sg[e] = k ? sg[e] + ag[j][e] : ag[j][e];
                        sb[e] = k ? sb[e] + ab[j][e] : ab[j][e];
                    }
                }
        }
    }
    __syncthreads();
    for (int64_t c = threadIdx.x; c < cols; c += BLOCK) {
        out[c] = comb[c];
        out[cols + c] = comb[pitch + c];
    }
}

// dgamma and dbeta from the blocks' sums: 32 columns a block, 16 rows of parts
// at a time.
__global__ void __launch_bounds__(512) ln_parts_kernel(const float *parts, int nparts, int wt, void *dgamma, void *dbeta,
                                                       int64_t cols) {
    __shared__ float sm[16][33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;  // of 2 * cols
    float s = 0.0f;
    if (c < 2 * cols)
        for (int i = w; i < nparts; i += 16) s += parts[(int64_t)i * 2 * cols + c];
    sm[w][lane] = s;
    __syncthreads();
    if (w == 0 && c < 2 * cols) {
#pragma unroll
        for (int i = 1; i < 16; i++) s += sm[i][lane];
        void *o = c < cols ? dgamma : dbeta;
        if (o) store_f(o, wt, c < cols ? c : c - cols, s);
    }
}

// Rows longer than the one-pass kernel holds: dx reads them twice, and the
// sums over rows read them again, 32 columns a block.
template <typename T>
__global__ void __launch_bounds__(1024) ln_dx_kernel(const T *dy, int64_t lddy, const T *x, int64_t ldx,
                                                     const float *mean, const float *rstd, int wt, const void *gamma,
                                                     T *dx, int64_t lddx, int64_t cols) {
    __shared__ float2 sm[32];
    const int64_t row = blockIdx.x;
    const T *xr = x + row * ldx, *dr = dy + row * lddy;
    T *o = dx + row * lddx;
    const float mu = mean[row], rs = rstd[row];
    float a = 0.0f, b = 0.0f;
    for (int64_t c = threadIdx.x; c < cols; c += 1024) {
        const float g = to_f(dr[c]) * (gamma ? load_f(gamma, wt, c) : 1.0f);
        a += g;
        b += g * ((to_f(xr[c]) - mu) * rs);
    }
    const float2 t = row_sum2<1024>(a, b, sm, 0);
    const float ma = t.x / (float)cols, mb = t.y / (float)cols;
    for (int64_t c = threadIdx.x; c < cols; c += 1024) {
        const float g = to_f(dr[c]) * (gamma ? load_f(gamma, wt, c) : 1.0f);
        o[c] = from_f<T>(rs * (g - ma - (to_f(xr[c]) - mu) * rs * mb));
    }
}
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

template <typename T>
int launch_grad_long(const T *dy, int64_t lddy, const T *x, int64_t ldx, const float *mean, const float *rstd, int wt,
                     const void *gamma, T *dx, int64_t lddx, void *dgamma, void *dbeta, int64_t rows, int64_t cols,
                     cudaStream_t s) {
    if (dgamma || dbeta) {  // before dx, which may take the place of dy or x
        ln_dw_kernel<T><<<(unsigned)((cols + 31) / 32), NT, 0, s>>>(dy, lddy, x, ldx, mean, rstd, wt, dgamma, dbeta, rows, cols);
        ZC_LAUNCHED("ln_dw_kernel");
    }
    if (dx && rows > 0) {
        ln_dx_kernel<T><<<(unsigned)rows, 1024, 0, s>>>(dy, lddy, x, ldx, mean, rstd, wt, gamma, dx, lddx, cols);
        ZC_LAUNCHED("ln_dx_kernel");
    }
    return ZPUCUDA_OK;
}

// Threads a row and rows a block of the one-pass gradient.
struct GradShape {
    int tpr, groups, blocks;
};
GradShape grad_shape(int64_t rows, int64_t cols) {
    GradShape g;
    g.tpr = cols <= 32 * kPerThread ? 32 : cols <= 256 * kPerThread ? 256 : cols <= 512 * kPerThread ? 512 : 1024;
    const int block = g.tpr == 32 ? 256 : g.tpr <= 512 ? 512 : 1024;
    g.groups = block / g.tpr;
    const int64_t want = (rows + g.groups - 1) / g.groups, most = (int64_t)num_sms() * (g.tpr == 32 ? kMaxParts : 1);
    g.blocks = (int)(want < most ? want : most);
    return g;
}

template <typename T, int TPR, int NV, int BLOCK>
int launch_grad(const GradShape &g, const T *dy, int64_t lddy, const T *x, int64_t ldx, const float *mean,
                const float *rstd, int wt, const void *gamma, T *dx, int64_t lddx, float *parts, int64_t rows,
                int64_t cols, cudaStream_t s) {
    auto f = ln_grad_kernel<T, TPR, NV, BLOCK>;
    const size_t smem = (size_t)((cols + kPiece<T> - 1) / kPiece<T> * kPiece<T>) * 8;
    if (smem > 40 * 1024) {  // at most 128 KiB
        static bool attr[64] = {false};
        const int dev = current_device();
        if (dev < 0 || dev >= 64 || !attr[dev]) {
            ZC_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, TPR * kPerThread * 8));
            if (dev >= 0 && dev < 64) attr[dev] = true;
        }
    }
    f<<<g.blocks, BLOCK, smem, s>>>(dy, lddy, x, ldx, mean, rstd, wt, gamma, dx, lddx, parts, rows, cols);
    ZC_LAUNCHED("ln_grad_kernel");
    return ZPUCUDA_OK;
}

template <typename T>
int launch_grad_for(const GradShape &g, const T *dy, int64_t lddy, const T *x, int64_t ldx, const float *mean,
                    const float *rstd, int wt, const void *gamma, T *dx, int64_t lddx, float *parts, int64_t rows,
                    int64_t cols, cudaStream_t s) {
#define GRAD(TPR, NV, BLOCK) \
    return launch_grad<T, TPR, NV, BLOCK>(g, dy, lddy, x, ldx, mean, rstd, wt, gamma, dx, lddx, parts, rows, cols, s)
    constexpr int NV = kPerThread / kPiece<T>;
    const bool half = cols * 2 <= (int64_t)g.tpr * kPerThread;  // half of the columns a thread
    if (g.tpr == 32) {
        if (half) GRAD(32, NV / 2, 256);
        GRAD(32, NV, 256);
    }
    if (g.tpr == 256) {
        if (half) GRAD(256, NV / 2, 512);
        GRAD(256, NV, 512);
    }
    if (g.tpr == 512) GRAD(512, NV, 512);
    GRAD(1024, NV, 1024);
#undef GRAD
}

}  // namespace
}  // namespace zc

using namespace zc;

extern "C" {

int zpucuda_layer_norm(int dtype, const void *d_x, int64_t ldx, int wtype, const void *d_gamma, const void *d_beta,
                       void *d_y, int64_t ldy, float *d_mean, float *d_rstd, int64_t rows, int64_t cols, double eps,
                       void *stream) {
    if (rows < 0 || cols < 1) return set_error(ZPUCUDA_ERR_INVALID_SHAPE, "layer_norm: rows >= 0 and cols >= 1 are wanted");
    if (rows > 0x7fffffff) return set_error(ZPUCUDA_ERR_NOT_SUPPORTED, "layer_norm: more than 2^31 - 1 rows");
    if (!(eps >= 0.0)) return set_error(ZPUCUDA_ERR_INVALID_ARGUMENT, "layer_norm: eps is negative or NaN");
    ZC_TRY(check_matrix("layer_norm", "x", d_x, dtype, ldx, rows, cols));
    ZC_TRY(check_matrix("layer_norm", "y", d_y, dtype, ldy, rows, cols));
    if (d_gamma) ZC_TRY(check_matrix("layer_norm", "gamma", d_gamma, wtype, cols, 1, cols));
    if (d_beta) ZC_TRY(check_matrix("layer_norm", "beta", d_beta, wtype, cols, 1, cols));
    if (rows == 0) return ZPUCUDA_OK;
    cudaStream_t s = resolve_stream(stream);
    ZC_HEAD_TYPE(dtype, T,
                 return launch_ln<T>((const T *)d_x, ldx, wtype, d_gamma, d_beta, (T *)d_y, ldy, d_mean, d_rstd, rows,
                                     cols, (float)eps, s));
}

int64_t zpucuda_layer_norm_grad_work(int64_t rows, int64_t cols) {
    if (rows < 0 || cols < 1 || cols > 1024 * kPerThread) return 0;
    return (int64_t)grad_shape(rows, cols).blocks * 2 * cols * (int64_t)sizeof(float);
}

int zpucuda_layer_norm_grad(int dtype, const void *d_dy, int64_t lddy, const void *d_x, int64_t ldx,
                            const float *d_mean, const float *d_rstd, int wtype, const void *d_gamma, void *d_dx,
                            int64_t lddx, void *d_dgamma, void *d_dbeta, int64_t rows, int64_t cols, void *d_work,
                            int64_t work_bytes, void *stream) {
    if (rows < 0 || cols < 1)
        return set_error(ZPUCUDA_ERR_INVALID_SHAPE, "layer_norm_grad: rows >= 0 and cols >= 1 are wanted");
    if (rows > 0x7fffffff) return set_error(ZPUCUDA_ERR_NOT_SUPPORTED, "layer_norm_grad: more than 2^31 - 1 rows");
    ZC_TRY(check_matrix("layer_norm_grad", "dy", d_dy, dtype, lddy, rows, cols));
    ZC_TRY(check_matrix("layer_norm_grad", "x", d_x, dtype, ldx, rows, cols));
    if (d_dx) ZC_TRY(check_matrix("layer_norm_grad", "dx", d_dx, dtype, lddx, rows, cols));
    if (d_gamma) ZC_TRY(check_matrix("layer_norm_grad", "gamma", d_gamma, wtype, cols, 1, cols));
    if (d_dgamma) ZC_TRY(check_matrix("layer_norm_grad", "dgamma", d_dgamma, wtype, cols, 1, cols));
    if (d_dbeta) ZC_TRY(check_matrix("layer_norm_grad", "dbeta", d_dbeta, wtype, cols, 1, cols));
    if (rows > 0 && (!d_mean || !d_rstd))
        return set_error(ZPUCUDA_ERR_INVALID_ARGUMENT, "layer_norm_grad: mean or rstd is null");
    const bool sums = d_dgamma || d_dbeta;
    const int64_t need = sums ? zpucuda_layer_norm_grad_work(rows, cols) : 0;
    if (need > 0 && (!d_work || work_bytes < need || !aligned_to(d_work, 16)))
        return set_error(ZPUCUDA_ERR_INVALID_ARGUMENT, "layer_norm_grad: work: null, too small or not 16-byte aligned");
    cudaStream_t s = resolve_stream(stream);
    if (cols > 1024 * kPerThread)
        ZC_HEAD_TYPE(dtype, T,
                     return launch_grad_long<T>((const T *)d_dy, lddy, (const T *)d_x, ldx, d_mean, d_rstd, wtype, d_gamma,
                                                (T *)d_dx, lddx, d_dgamma, d_dbeta, rows, cols, s));
    const GradShape g = grad_shape(rows, cols);
    if (rows > 0 && (d_dx || sums)) {
        ZC_HEAD_TYPE(dtype, T,
                     ZC_TRY(launch_grad_for<T>(g, (const T *)d_dy, lddy, (const T *)d_x, ldx, d_mean, d_rstd, wtype,
                                               d_gamma, (T *)d_dx, lddx, sums ? (float *)d_work : nullptr, rows, cols, s)));
    }
    if (sums) {
        ln_parts_kernel<<<(unsigned)((2 * cols + 31) / 32), 512, 0, s>>>((const float *)d_work, rows > 0 ? g.blocks : 0, wtype,
                                                                        d_dgamma, d_dbeta, cols);
        ZC_LAUNCHED("ln_parts_kernel");
    }
    return ZPUCUDA_OK;
}

}  // extern "C"
