// Layer norm over the last axis, forward and backward (nn.layerNorm,
// restated for a batch of rows):
//   mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps)
//   y = (x - mu) * rstd * gamma + beta
// and with xhat = (x - mu) * rstd, g = dy * gamma:
//   dx = rstd * (g - mean(g) - xhat * mean(g * xhat))
//   dgamma = sum over rows of dy * xhat,  dbeta = sum over rows of dy.
// HBM bounds both: a row is read once into registers, reduced there, and
// written.  What keeps them from its rate are the two sums of a row that
// everything waits for: rows are on their way to shared memory meanwhile, and a
// row is held by few threads.  Forward 16384 x 1024 f16 takes 14.0 us (4.8 TB/s),
// 4096 x 4096 bf16 15.0 us, 4 x 4096 2.8 us; backward 8192 x 4096 bf16 44 us
// (4.6 TB/s), 1021 x 5003 f32 26.3 us (2.3 TB/s: pieces off the 16-byte grid are
// shifted into place on both ways).  The gradient's blocks walk rows and keep their columns' sums of
// dgamma and dbeta in registers; one row of sums a block goes to the caller's
// workspace, and a second kernel adds those up in the blocks' order, so a
// result does not depend on the run.
#include "head.cuh"

namespace zc {
namespace {

constexpr int NT = 256;
constexpr int kPerThread = 16;  // columns of a row that a thread of the gradient holds
constexpr int kMaxCluster = 8;  // blocks of a cluster of it
// What lies before a row that is not among a block's first D: more than a granule.  Rows shorter than a granule are taken
// by blocks of 8 rows with D = 4, so 32 of them lie before it.
constexpr int64_t kInside = INT64_MAX;
constexpr int64_t kMaxOnePass = 512 * kPerThread * kMaxCluster;

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
// sm: 2 * TPR / 32 floats of the row's own; barrier `bar` is the row's own.
template <int TPR>
__device__ __forceinline__ float2 row_sum2(float a, float b, float *sm, int bar) {
    const int lane = threadIdx.x & 31;
    const bool up = lane & 16;  // the lower lanes go on with a, the upper ones with b
    float v = (up ? b : a) + __shfl_xor_sync(0xffffffffu, up ? a : b, 16);
#pragma unroll
    for (int o = 8; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (TPR > 32) {
        constexpr int W = TPR / 32;
        if ((lane & 15) == 0) sm[((threadIdx.x % TPR) >> 5) + (up ? W : 0)] = v;
        asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(TPR) : "memory");
        if constexpr (W == 32) {
            float p = sm[lane], q = sm[32 + lane];
            v = (up ? q : p) + __shfl_xor_sync(0xffffffffu, up ? p : q, 16);
#pragma unroll
            for (int o = 8; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        } else {
            v = sm[(lane & (W - 1)) + (up ? W : 0)];
#pragma unroll
            for (int o = W / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        }
    }
    return make_float2(__shfl_sync(0xffffffffu, v, 0), __shfl_sync(0xffffffffu, v, 16));
}

// ------------------------------------------------------------------ forward

// The weights of a piece in pairs.
template <int N>
__device__ __forceinline__ void load_w2(const void *p, int wt, int64_t i, int have, float dflt, f32x2 (&f)[N / 2]) {
    float w[N];
    load_w<N>(p, wt, i, have, dflt, w);
#pragma unroll
    for (int e = 0; e < N / 2; e++) f[e] = make2(w[2 * e], w[2 * e + 1]);
}

// What a thread does with its pieces of a row, forward.  The mean of what the
// rounded mean leaves (`rest`) is taken off again: rows far from zero keep the
// digits that a 32-bit mean alone would cost them.
template <typename T>
struct Fwd {
    static constexpr int N = kPiece<T>, H = N / 2;
    static __device__ __forceinline__ void sum(const f32x2 (&a)[H], f32x2 &s) {  // what is past the row's end is 0
#pragma unroll
        for (int e = 0; e < H; e++) s = add2(s, a[e]);
    }
    static __device__ __forceinline__ void spread(f32x2 (&a)[H], int have, float mu, f32x2 &d1, f32x2 &d2) {
#pragma unroll
        for (int e = 0; e < H; e++) {
            a[e] = add2(a[e], make2(-mu));
            if (have < N && 2 * e + 1 >= have) a[e] = make2(2 * e < have ? lo2(a[e]) : 0.0f, 0.0f);
            d1 = add2(d1, a[e]);
            d2 = fma2(a[e], a[e], d2);
        }
    }
    // (mean - mu, 1 / deviation) from the sums of d and d^2.
    static __device__ __forceinline__ float2 finish(float2 q, float inv, float eps) {
        const float rest = q.x * inv;
        float var = q.y * inv - rest * rest;
        var = var < 0.0f ? 0.0f : var;  // NaN stays
        return make_float2(rest, 1.0f / sqrtf(var + eps));
    }
    static __device__ __forceinline__ uint4 out(const f32x2 (&a)[H], float2 f, const f32x2 (&g)[H], const f32x2 (&b)[H]) {
        f32x2 y[H];
#pragma unroll
        for (int e = 0; e < H; e++) y[e] = fma2(mul2(add2(a[e], make2(-f.x)), make2(f.y)), g[e], b[e]);
        return pack2<T>(y);
    }
};

// TPR threads a row, NV pieces a thread, whose weights it keeps in registers; a
// block walks rows, D of them on their way to shared memory while one is worked on.
template <typename T, int TPR, int NV, int D, bool EVEN>
__global__ void __launch_bounds__(TPR < NT ? NT : TPR)
    ln_kernel(const T *x, int64_t ldx, int wt, const void *gamma, const void *beta, T *y, int64_t ldy, float *mean,
              float *rstd, int64_t rows, int64_t cols, float eps) {
    constexpr int BLOCK = TPR < NT ? NT : TPR, GROUPS = BLOCK / TPR, N = kPiece<T>;
    extern __shared__ uint4 ring_smem[];
    __shared__ float sm[2][2][BLOCK / 16];
    const int t = threadIdx.x % TPR, group = threadIdx.x / TPR, bar = 1 + (TPR > 32 ? group : 0);
    const int p0 = (t >> 5) * (32 * NV) + (t & 31);  // its first piece
    const RowRing<T, NV, 1, D, EVEN> ring(ring_smem, p0);
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    int64_t row = (int64_t)blockIdx.x * GROUPS + group;
    const float inv = 1.0f / (float)cols;
#pragma unroll
    for (int d = 0; d < D; d++) {
        if (row + d * step < rows) ring.issue(d, 0, x + (row + d * step) * ldx, cols, (row + d * step) * ldx);
        ring.commit();
    }
    f32x2 g[NV][N / 2], b[NV][N / 2];
    int have[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        have[j] = EVEN ? ((int64_t)(p0 + j * 32) * N < cols ? N : 0) : in_row<N>(p0 + j * 32, cols);
        load_w2<N>(gamma, wt, p0 + j * 32, have[j], 1.0f, g[j]);
        load_w2<N>(beta, wt, p0 + j * 32, have[j], 0.0f, b[j]);
    }
    int slot = 0;
    for (int odd = 0; row < rows; row += step, odd ^= 1) {
        ring.wait();
        f32x2 v[NV][N / 2], s = make2(0.0f), d1 = s, d2 = s;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            unpack2<T>(ring.read(slot, 0, j, x + row * ldx, cols), v[j]);
            Fwd<T>::sum(v[j], s);
        }
        __syncwarp();
        if (row + D * step < rows) ring.issue(slot, 0, x + (row + D * step) * ldx, cols, kInside);
        ring.commit();
        slot = slot + 1 == D ? 0 : slot + 1;
        const float mu = row_sum2<TPR>(lo2(s) + hi2(s), 0.0f, sm[odd][0] + group * (TPR / 16), bar).x * inv;
#pragma unroll
        for (int j = 0; j < NV; j++)
            if (!EVEN || have[j]) Fwd<T>::spread(v[j], EVEN ? N : have[j], mu, d1, d2);
        const float2 f = Fwd<T>::finish(row_sum2<TPR>(lo2(d1) + hi2(d1), lo2(d2) + hi2(d2), sm[odd][1] + group * (TPR / 16), bar), inv, eps);
        T *yr = y + row * ldy;
        uint4 o[NV];
#pragma unroll
        for (int j = 0; j < NV; j++) {
            o[j] = Fwd<T>::out(v[j], f, g[j], b[j]);
            if (EVEN && have[j]) *(uint4 *)(yr + (p0 + j * 32) * N) = o[j];
        }
        if constexpr (!EVEN) {
            __syncwarp();
            store_run<T, NV>(yr, p0, (int)cols, o);
        }
        if (t == 0) {
            if (mean) mean[row] = mu + f.x;
            if (rstd) rstd[row] = f.y;
        }
    }
}

// Rows too long for the above: read three times, from L2 after the first.
template <typename T>
__global__ void __launch_bounds__(1024)
    ln_long_kernel(const T *x, int64_t ldx, int wt, const void *gamma, const void *beta, T *y, int64_t ldy, float *mean,
                   float *rstd, int64_t cols, float eps) {
    constexpr int N = kPiece<T>;
    __shared__ float sm[2][64];
    const int64_t row = blockIdx.x, n = (cols + N - 1) / N;
    const T *xr = x + row * ldx;
    const float inv = 1.0f / (float)cols;
    f32x2 v[N / 2], s = make2(0.0f), d1 = s, d2 = s;
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
        unpack2<T>(load_piece(xr, i, cols), v);
        Fwd<T>::sum(v, s);
    }
    const float mu = row_sum2<1024>(lo2(s) + hi2(s), 0.0f, sm[0], 1).x * inv;
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
        unpack2<T>(load_piece(xr, i, cols), v);
        Fwd<T>::spread(v, in_row<N>(i, cols), mu, d1, d2);
    }
    const float2 f = Fwd<T>::finish(row_sum2<1024>(lo2(d1) + hi2(d1), lo2(d2) + hi2(d2), sm[1], 1), inv, eps);
    for (int64_t i = threadIdx.x; i - (threadIdx.x & 31) < n; i += 1024) {
        f32x2 none = make2(0.0f), unused = none;
        unpack2<T>(i < n ? load_piece(xr, i, cols) : make_uint4(0, 0, 0, 0), v);
        Fwd<T>::spread(v, in_row<N>(i, cols), mu, none, unused);
        f32x2 g[N / 2], b[N / 2];
        load_w2<N>(gamma, wt, i, in_row<N>(i, cols), 1.0f, g);
        load_w2<N>(beta, wt, i, in_row<N>(i, cols), 0.0f, b);
        const uint4 o = Fwd<T>::out(v, f, g, b);
        __syncwarp();
        store_piece(y + row * ldy, i, cols, o);
    }
    if (threadIdx.x == 0) {
        if (mean) mean[row] = mu + f.x;
        if (rstd) rstd[row] = f.y;
    }
}

// Whether rows of cols elements at pitches of ld start on 16-byte boundaries and hold whole pieces.
template <typename T>
bool even_rows(const void *p, int64_t ld, int64_t rows, int64_t cols) {
    return cols % kPiece<T> == 0 && aligned_to(p, 16) && (rows <= 1 || ld % kPiece<T> == 0);
}

template <typename T, int TPR, int NV, int D, bool EVEN>
int launch_ln_ring(const T *x, int64_t ldx, int wt, const void *gamma, const void *beta, T *y, int64_t ldy, float *mean,
                   float *rstd, int64_t rows, int64_t cols, float eps, cudaStream_t s) {
    constexpr int BLOCK = TPR < NT ? NT : TPR, GROUPS = BLOCK / TPR;
    auto f = ln_kernel<T, TPR, NV, D, EVEN>;
    const size_t smem = (size_t)(BLOCK / 32) * RowRing<T, NV, 1, D, EVEN>::kWarp * 16;
    static int cache[64] = {0};
    const int per = blocks_per_sm(f, BLOCK, smem, smem, cache);
    if (!per) return cuda_fail(cudaGetLastError(), "layer_norm: occupancy");
    const int64_t want = (rows + GROUPS - 1) / GROUPS, most = (int64_t)per * num_sms();
    f<<<(unsigned)(want < most ? want : most), BLOCK, smem, s>>>(x, ldx, wt, gamma, beta, y, ldy, mean, rstd, rows, cols, eps);
    ZC_LAUNCHED("ln_kernel");
    return ZPUCUDA_OK;
}

template <typename T>
int launch_ln(const T *x, int64_t ldx, int wt, const void *gamma, const void *beta, T *y, int64_t ldy, float *mean,
              float *rstd, int64_t rows, int64_t cols, float eps, cudaStream_t s) {
    const int64_t n = (cols + kPiece<T> - 1) / kPiece<T>;
    const bool even = even_rows<T>(x, ldx, rows, cols) && even_rows<T>(y, ldy, rows, cols);
#define LN(...)                                                                                                              \
    return even ? launch_ln_ring<T, __VA_ARGS__, true>(x, ldx, wt, gamma, beta, y, ldy, mean, rstd, rows, cols, eps, s)      \
                : launch_ln_ring<T, __VA_ARGS__, false>(x, ldx, wt, gamma, beta, y, ldy, mean, rstd, rows, cols, eps, s)
    // Four pieces a thread, and as few threads a row as hold it: sums over few warps cost the least.  (16384 x 1024 f16:
    // 14.6 us with 32 threads, 16.9 with 64, 20.2 with 128; 4096 x 4096 bf16 15.7 with 128, 20.6 with 512.)  Fewer pieces
    // for rows that would leave most lanes without: 16384 x 102 bf16 10.2 us with one, 15.9 with two.
    // 16-bit rows above 16384 columns do not fit 1024 threads' registers this way (1.4 to 1.8 KB of spills a thread: 1024 x
    // 32768 bf16 116 us, 2048 x 16384 28).
    if (n <= 32) LN(32, 1, 4);
    if (n <= 64) LN(32, 2, 3);
    if (n <= 128) LN(32, 4, 2);
    if (n <= 256) LN(64, 4, 2);
    if (n <= 512) LN(128, 4, 2);
    if (n <= 1024) LN(256, 4, 2);
    if (n <= 2048) LN(512, 4, 2);
    if (n <= 4096) LN(1024, 4, 2);
#undef LN
    ln_long_kernel<T><<<(unsigned)rows, 1024, 0, s>>>(x, ldx, wt, gamma, beta, y, ldy, mean, rstd, cols, eps);
    ZC_LAUNCHED("ln_long_kernel");
    return ZPUCUDA_OK;
}

// ----------------------------------------------------------------- backward

// One pass: TPR threads a row, BLOCK / TPR rows of a block at a time, NV pieces a
// thread; D rows are on their way to shared memory while one is worked on.  A row
// that a block does not hold is split over a cluster (CLUSTER), whose blocks tell
// one another their parts of its two sums.  parts: a row of [2][cols] sums for
// each block (cluster), or null.
template <typename T, int TPR, int NV, int BLOCK, int D, bool CLUSTER, bool EVEN>
__global__ void __launch_bounds__(BLOCK)
    ln_grad_kernel(const T *dy, int64_t lddy, const T *x, int64_t ldx, const float *mean, const float *rstd, int wt,
                   const void *gamma, T *dx, int64_t lddx, float *parts, int64_t rows, int64_t cols) {
    constexpr int GROUPS = BLOCK / TPR, N = kPiece<T>, PITCH = TPR * NV * N;
    __shared__ float2 peers[2][kMaxCluster];
    __shared__ float sm[2][BLOCK / 16];
    extern __shared__ uint4 grad_smem[];
    uint32_t rank = 0, size = 1;
    if constexpr (CLUSTER) {
        asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // this block runs
    }
    const int group = threadIdx.x / TPR, bar = 1 + (TPR > 32 ? group : 0);
    const int t = threadIdx.x % TPR, t0 = (t >> 5) * (32 * NV) + (t & 31);
    const int p0 = t0 + (int)rank * TPR * NV;  // its first piece, of the block's part of a row (t0) and of the row
    const int64_t n = (cols + N - 1) / N;
    const float inv = 1.0f / (float)cols;
    f32x2 g[NV][N / 2], ag[NV][N / 2], ab[NV][N / 2];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        load_w2<N>(gamma, wt, p0 + j * 32, in_row<N>(p0 + j * 32, cols), 1.0f, g[j]);
#pragma unroll
        for (int e = 0; e < N / 2; e++) ag[j][e] = ab[j][e] = make2(0.0f);
    }
    const RowRing<T, NV, 2, D, EVEN> ring(grad_smem, p0);
    const int64_t step = (int64_t)(gridDim.x / size) * GROUPS;
    int64_t row = (int64_t)(blockIdx.x / size) * GROUPS + group;
    auto issue = [&](int slot, int64_t r, auto later) {
        if (r < rows) {
            ring.issue(slot, 0, x + r * ldx, cols, decltype(later)::value ? kInside : r * ldx);
            ring.issue(slot, 1, dy + r * lddy, cols, decltype(later)::value ? kInside : r * lddy);
        }
        ring.commit();
    };
#pragma unroll
    for (int d = 0; d < D; d++) issue(d, row + d * step, std::false_type());
    int slot = 0;
    float next_mu = 0.0f, next_rs = 0.0f;
    if (row < rows) {
        next_mu = mean[row];
        next_rs = rstd[row];
    }
    // no block writes to another's shared memory before that one runs
    if constexpr (CLUSTER) {
        __syncwarp();
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    for (int odd = 0; row < rows; row += step, odd ^= 1) {
        const float mu = next_mu, rs = next_rs;
        if (row + step < rows) {
            next_mu = mean[row + step];
            next_rs = rstd[row + step];
        }
        ring.wait();
        // xhat and dy * gamma; past the row's end dy is 0, and all that follows from it
        f32x2 xh[NV][N / 2], gd[NV][N / 2], a = make2(0.0f), b = a;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            f32x2 d[N / 2];
            unpack2<T>(ring.read(slot, 0, j, x + row * ldx, cols), xh[j]);
            unpack2<T>(ring.read(slot, 1, j, dy + row * lddy, cols), d);
#pragma unroll
            for (int e = 0; e < N / 2; e++) {
                xh[j][e] = mul2(add2(xh[j][e], make2(-mu)), make2(rs));
                gd[j][e] = mul2(d[e], g[j][e]);
                a = add2(a, gd[j][e]);
                b = fma2(gd[j][e], xh[j][e], b);
                ag[j][e] = fma2(d[e], xh[j][e], ag[j][e]);
                ab[j][e] = add2(ab[j][e], d[e]);
            }
        }
        __syncwarp();
        issue(slot, row + D * step, std::true_type());
        slot = slot + 1 == D ? 0 : slot + 1;
        if (!dx) continue;
        // two buffers: a thread that is a row ahead does not overwrite what another still reads
        float2 q = row_sum2<TPR>(lo2(a) + hi2(a), lo2(b) + hi2(b), sm[odd] + group * (TPR / 16), bar);
        if constexpr (CLUSTER) {
            if (threadIdx.x < size) {
                uint32_t there;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                             : "=r"(there)
                             : "r"((uint32_t)__cvta_generic_to_shared(&peers[odd][rank])), "r"(threadIdx.x));
                asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(there), "f"(q.x), "f"(q.y) : "memory");
            }
            __syncwarp();
            asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
            q = make_float2(0.0f, 0.0f);
            for (uint32_t r = 0; r < size; r++) {
                q.x += peers[odd][r].x;
                q.y += peers[odd][r].y;
            }
        }
        const f32x2 m = make2(-rs * (q.x * inv)), k = make2(-rs * (q.y * inv)), r2 = make2(rs);
        T *out = dx + row * lddx;
        uint4 o[NV];
#pragma unroll
        for (int j = 0; j < NV; j++) {
#pragma unroll
            for (int e = 0; e < N / 2; e++) xh[j][e] = fma2(xh[j][e], k, fma2(gd[j][e], r2, m));
            o[j] = pack2<T>(xh[j]);
            if (EVEN && p0 + j * 32 < n) *(uint4 *)(out + (p0 + j * 32) * N) = o[j];
        }
        if constexpr (!EVEN) {
            __syncwarp();
            store_run<T, NV>(out, p0, (int)cols, o);
        }
    }
    // no block ends while another may still write to its shared memory
    if constexpr (CLUSTER) {
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    if (!parts) return;
    // the groups add up in their order, in the ring's place
    asm volatile("cp.async.wait_all;" ::: "memory");
    float *comb = (float *)grad_smem;  // [2][PITCH]
    for (int k = 0; k < GROUPS; k++) {
        __syncthreads();
        if (group == k)
#pragma unroll
            for (int j = 0; j < NV; j++) {
                float *sg = comb + (t0 + j * 32) * N, *sb = sg + PITCH;
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const float u = e & 1 ? hi2(ag[j][e / 2]) : lo2(ag[j][e / 2]), v = e & 1 ? hi2(ab[j][e / 2]) : lo2(ab[j][e / 2]);
                    sg[e] = k ? sg[e] + u : u;
                    sb[e] = k ? sb[e] + v : v;
                }
            }
    }
    __syncthreads();
    const int64_t c0 = (int64_t)rank * PITCH, m = cols - c0 < PITCH ? cols - c0 : PITCH;
    float *out = parts + (int64_t)(blockIdx.x / size) * 2 * cols + c0;
    for (int64_t c = threadIdx.x; c < m; c += BLOCK) {
        out[c] = comb[c];
        out[cols + c] = comb[PITCH + c];
    }
}

// dgamma and dbeta from the blocks' sums: 32 columns a block, 16 rows of parts
// at a time.  It may be launched while the kernel that makes the sums still runs,
// and waits for its end.
__global__ void __launch_bounds__(512) ln_parts_kernel(const float *parts, int nparts, int wt, void *dgamma, void *dbeta,
                                                       int64_t cols) {
    __shared__ float sm[16][33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;  // of 2 * cols
    float s = 0.0f;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (c < 2 * cols) {
        const float *p = parts + c;
        for (int i = w; i < nparts; i += 160) {  // ten loads in flight
            float v[10];
#pragma unroll
            for (int u = 0; u < 10; u++) v[u] = i + 16 * u < nparts ? p[(int64_t)(i + 16 * u) * 2 * cols] : 0.0f;
#pragma unroll
            for (int u = 0; u < 10; u++) s += v[u];
        }
    }
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
    __shared__ float sm[64];
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
    const float2 t = row_sum2<1024>(a, b, sm, 1);
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

// Threads a row, rows a block, blocks a row and rows of sums of the one-pass gradient.  As few threads as hold the row (16384
// x 1024 f16: 30 us with 64, 54 with 256), and blocks of 512, which fill the registers: more that keep less were slower.
struct GradShape {
    int tpr, groups, cluster, parts;
};
GradShape grad_shape(int64_t rows, int64_t cols) {
    GradShape g;
    g.tpr = 32;
    while (g.tpr < 512 && cols > (int64_t)g.tpr * kPerThread) g.tpr *= 2;
    g.groups = (g.tpr == 32 ? 256 : 512) / g.tpr;
    g.cluster = (int)((cols + (int64_t)g.tpr * kPerThread - 1) / ((int64_t)g.tpr * kPerThread));
    const int64_t want = (rows + g.groups - 1) / g.groups, most = (int64_t)num_sms() * (g.tpr == 32 ? 2 : 1) / g.cluster;
    g.parts = (int)(want < most ? want : most);
    return g;
}

template <typename T, int TPR, int NV, int BLOCK, int D, bool CLUSTER, bool EVEN>
int launch_grad(const GradShape &g, const T *dy, int64_t lddy, const T *x, int64_t ldx, const float *mean,
                const float *rstd, int wt, const void *gamma, T *dx, int64_t lddx, float *parts, int64_t rows,
                int64_t cols, cudaStream_t s) {
    auto f = ln_grad_kernel<T, TPR, NV, BLOCK, D, CLUSTER, EVEN>;
    // the ring, in whose place the sums are added up at the end
    constexpr size_t ring = (size_t)(BLOCK / 32) * RowRing<T, NV, 2, D, EVEN>::kWarp * 16, sums = (size_t)TPR * NV * kPiece<T> * 8;
    constexpr size_t smem = ring > sums ? ring : sums;
    static_assert(smem <= 226 * 1024, "shared memory");
    static int cache[64] = {0};
    if (!blocks_per_sm(f, BLOCK, smem, smem, cache)) return cuda_fail(cudaGetLastError(), "layer_norm_grad: occupancy");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(g.parts * g.cluster));
    cfg.blockDim = dim3(BLOCK);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1] = {};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)g.cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = CLUSTER ? 1 : 0;
    ZC_CUDA(cudaLaunchKernelEx(&cfg, f, dy, lddy, x, ldx, mean, rstd, wt, gamma, dx, lddx, parts, rows, cols));
    count_launch();
    return ZPUCUDA_OK;
}

template <typename T>
int launch_grad_for(const GradShape &g, const T *dy, int64_t lddy, const T *x, int64_t ldx, const float *mean,
                    const float *rstd, int wt, const void *gamma, T *dx, int64_t lddx, float *parts, int64_t rows,
                    int64_t cols, cudaStream_t s) {
    constexpr int NV = kPerThread / kPiece<T>, D = NV > 2 ? 2 : 4;
    const bool even = even_rows<T>(x, ldx, rows, cols) && even_rows<T>(dy, lddy, rows, cols) && even_rows<T>(dx, lddx, rows, cols);
#define GRAD(...)                                                                                                                     \
    return even ? launch_grad<T, __VA_ARGS__, true>(g, dy, lddy, x, ldx, mean, rstd, wt, gamma, dx, lddx, parts, rows, cols, s)       \
                : launch_grad<T, __VA_ARGS__, false>(g, dy, lddy, x, ldx, mean, rstd, wt, gamma, dx, lddx, parts, rows, cols, s)
    if (cols <= 16 * kPerThread) GRAD(32, NV / 2, 256, 4, false);
    if (g.tpr == 32) GRAD(32, NV, 256, 4, false);
    if (g.tpr == 64) GRAD(64, NV, 512, D, false);
    if (g.tpr == 128) GRAD(128, NV, 512, D, false);
    if (g.tpr == 256) GRAD(256, NV, 512, D, false);
    if (g.cluster == 1) GRAD(512, NV, 512, D, false);
    GRAD(512, NV, 512, D, true);
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
    ZC_TRY(check_vectors("layer_norm", 4, {{"mean", d_mean}, {"rstd", d_rstd}}));
    if (rows == 0) return ZPUCUDA_OK;
    cudaStream_t s = resolve_stream(stream);
    ZC_HEAD_TYPE(dtype, T,
                 return launch_ln<T>((const T *)d_x, ldx, wtype, d_gamma, d_beta, (T *)d_y, ldy, d_mean, d_rstd, rows,
                                     cols, (float)eps, s));
}

int64_t zpucuda_layer_norm_grad_work(int64_t rows, int64_t cols) {
    if (rows < 0 || cols < 1 || cols > kMaxOnePass) return 0;
    return (int64_t)grad_shape(rows, cols).parts * 2 * cols * (int64_t)sizeof(float);
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
    ZC_TRY(check_vectors("layer_norm_grad", 4, {{"mean", d_mean}, {"rstd", d_rstd}}));
    if (rows > 0 && (!d_mean || !d_rstd))
        return set_error(ZPUCUDA_ERR_INVALID_ARGUMENT, "layer_norm_grad: mean or rstd is null");
    const bool sums = d_dgamma || d_dbeta;
    const int64_t need = sums ? zpucuda_layer_norm_grad_work(rows, cols) : 0;
    if (need > 0 && (!d_work || work_bytes < need || !aligned_to(d_work, 16)))
        return set_error(ZPUCUDA_ERR_INVALID_ARGUMENT, "layer_norm_grad: work: null, too small or not 16-byte aligned");
    cudaStream_t s = resolve_stream(stream);
    if (cols > kMaxOnePass)
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
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)((2 * cols + 31) / 32));
        cfg.blockDim = dim3(512);
        cfg.stream = s;
        cudaLaunchAttribute at[1] = {};
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = at;
        cfg.numAttrs = rows > 0 ? 1 : 0;
        ZC_CUDA(cudaLaunchKernelEx(&cfg, ln_parts_kernel, (const float *)d_work, rows > 0 ? g.parts : 0, wtype, d_dgamma,
                                   d_dbeta, cols));
        count_launch();
    }
    return ZPUCUDA_OK;
}

}  // extern "C"
