// The linear layer in 8-bit integers: rows quantised with one scale each,
//   scale = max |x| / 127,  q = round-half-to-even(x / scale)
// (a row of zeros keeps scale 0; a row with a NaN or an infinity gets scale
// NaN and q = 0, so only its own outputs become NaN), and the product
//   y[m, n] = (sum over k of a[m, k] * b[n, k]) * sa[m] * sb[n] + bias[n]
// whose sum is exact in 32-bit integers.
#include <string.h>

#include "head.cuh"
#include "int8.cuh"
#include "tcgen05.cuh"

namespace zc {

static __device__ unsigned int g_int8_error;

int int8_device_error(unsigned int *e) {
    ZC_CUDA(cudaMemcpyFromSymbol(e, g_int8_error, sizeof *e));
    return ZPUCUDA_OK;
}

namespace {

constexpr int NT = 256;
// 131071 * 128 * 128 < 2^31: no sum of that many products leaves 32 bits.
constexpr int64_t kMaxInner = 131071;

// One result from its sum, rounded alike on every path.
__device__ __forceinline__ float result(int sum, float sa, float sb, const float *bias, float b) {
    const float v = __fmul_rn(__fmul_rn((float)sum, sa), sb);
    return bias ? __fadd_rn(v, b) : v;
}

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
            if (r < m && c < n) out[r * ldo + c] = from_f<T>(result(acc[i][j], sa[r], sb[c], bias, bias ? bias[c] : 0.0f));
        }
}

// A product on the tensor cores: D[p, q] = sum over k of P[p, k] * Q[q, k] in
// tiles of 128 x BN, for operands that a tensor map can describe (addresses
// and row pitches multiples of 16 bytes).  P is a and Q is b, or (SWAP) P is b
// and Q is a: with few tokens the weights fill the 128 rows and a narrow tile
// holds the tokens, so no multiplication is spent on rows that are not there.
//
// One CTA per SM walks tiles; warp 0 loads 128-byte slices of both operands by
// TMA into a ring of stages, one lane of warp 1 issues tcgen05.mma (kind::i8,
// exact 32-bit sums in TMEM), warps 2-5 turn a finished tile into the result
// while the next one is summed into the other TMEM buffer.  With few tiles the
// inner axis is split over a cluster, whose CTAs hand their sums to the first
// through shared memory (whole numbers: the split does not change the result).
constexpr int TC_THREADS = 192;
constexpr int TC_STAGE_A = 128 * 128;
template <int BN>
struct TcTile {
    static constexpr int STAGE = TC_STAGE_A + BN * 128;
    static constexpr int STAGES = BN == 256 ? 4 : BN == 128 ? 6 : 8;
    static constexpr int COLS = 2 * BN < 32 ? 32 : 2 * BN;  // two sums in TMEM
    static constexpr int PART = 128 * (BN + 1) * 4;         // a split's sums, rows padded against bank conflicts
    static constexpr int XPOSE = 4 * 32 * 33 * 4;           // 32 x 32 results of each of the four storing warps
    static constexpr int SMEM = STAGES * STAGE + XPOSE + 1024;
    static_assert(SMEM <= 227 * 1024 && (BN == 256 || PART <= STAGES * STAGE), "shared memory");
};

struct TcArgs {
    const float *sa, *sb, *bias;  // by token, by channel
    void *out;
    int64_t ldo, tokens, channels;
    int tiles_p, tiles_q, group;  // tiles along P and Q; P tiles per raster group
    int kt, kt_split, splits;     // 128-byte slices, slices of a split
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ const void *cluster_map(const void *p, uint32_t rank) {
    uint64_t r;
    asm volatile("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"((uint64_t)p), "r"(rank));
    return (const void *)r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int BN, bool SWAP, typename T>
__global__ void __launch_bounds__(TC_THREADS, 1)
    int8_tc_kernel(const __grid_constant__ CUtensorMap mp, const __grid_constant__ CUtensorMap mq, const TcArgs A) {
    using TT = TcTile<BN>;
    extern __shared__ uint8_t raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[TT::STAGES], empty[TT::STAGES], tfull[2], tfree[2];
    __shared__ uint32_t tmem_base;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ntiles = A.tiles_p * A.tiles_q;
    const int split = A.splits > 1 ? (int)cluster_rank() : 0;
    const int k0 = split * A.kt_split, k1 = min(A.kt, k0 + A.kt_split);
    // tile t: P tiles run fastest inside a group of A.group of them, so that the
    // tiles in flight together share operand rows in L2
    auto place = [&](int t, int *tp, int *tq) {
        const int per = A.group * A.tiles_q, g = t / per, first = g * A.group;
        const int rows = min(A.group, A.tiles_p - first);
        *tp = first + (t - g * per) % rows;
        *tq = (t - g * per) / rows;
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < TT::STAGES; s++) {
            tc::mb_init(&full[s], 1);
            tc::mb_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            tc::mb_init(&tfull[b], 1);
            tc::mb_init(&tfree[b], 128);
        }
        tc::mb_init_fence();
    }
    if (warp == 1) tc::tmem_alloc(&tmem_base, TT::COLS);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_base;

    if (warp == 0) {
        if (lane == 0) {
            int j = 0;  // slices issued
            bool ok = true;
            for (int t = blockIdx.x; t < ntiles && ok; t += gridDim.x) {
                int tp, tq;
                place(t, &tp, &tq);
                for (int k = k0; k < k1; k++, j++) {
                    const int s = j % TT::STAGES;
                    if (j >= TT::STAGES && !tc::mb_wait(&empty[s], ((j / TT::STAGES) - 1) & 1, &g_int8_error)) {
                        ok = false;
                        break;
                    }
                    uint8_t *st = smem + s * TT::STAGE;
                    tc::mb_expect_tx(&full[s], TT::STAGE);
                    tc::tma_load_2d(st, &mp, k * 128, tp * 128, &full[s]);
                    tc::tma_load_2d(st + TC_STAGE_A, &mq, k * 128, tq * BN, &full[s]);
                }
            }
            if (!ok)  // give up only once the copies in flight have landed
                for (int i = max(0, j - TT::STAGES); i < j; i++)
                    tc::mb_wait(&full[i % TT::STAGES], (i / TT::STAGES) & 1, &g_int8_error);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t ID = tc::idesc_s8(128, BN);
            int j = 0, n = 0;
            bool ok = true;
            for (int t = blockIdx.x; t < ntiles && ok; t += gridDim.x, n++) {
                const int buf = n & 1;
                if (n >= 2 && !tc::mb_wait(&tfree[buf], ((n >> 1) - 1) & 1, &g_int8_error)) break;
                tc::fence_after();
                for (int k = k0; k < k1; k++, j++) {
                    const int s = j % TT::STAGES;
                    if (!tc::mb_wait(&full[s], (j / TT::STAGES) & 1, &g_int8_error)) {
                        ok = false;
                        break;
                    }
                    tc::fence_after();
                    const uint8_t *st = smem + s * TT::STAGE;
#pragma unroll
                    for (int kk = 0; kk < 4; kk++)
                        tc::mma_s8(tmem + buf * BN, tc::desc_k128(st + kk * 32), tc::desc_k128(st + TC_STAGE_A + kk * 32),
                                   ID, k > k0 || kk > 0);
                    tc::mma_commit(&empty[s]);
                }
                if (ok) tc::mma_commit(&tfull[buf]);
            }
        }
    } else {
        const int q4 = warp & 3;  // the quarter of the TMEM lanes that this warp may read
        const uint32_t lanes = (uint32_t)(q4 * 32) << 16;
        T *out = (T *)A.out;
        float *turn = (float *)(smem + TT::STAGES * TT::STAGE) + q4 * 32 * 33;
        const bool vec = !SWAP && ((uintptr_t)out & 15) == 0 && (A.ldo * (int64_t)sizeof(T)) % 16 == 0;
        int n = 0;
        for (int t = blockIdx.x; t < ntiles; t += gridDim.x, n++) {
            int tp, tq;
            place(t, &tp, &tq);
            const int buf = n & 1;
            if (!tc::mb_wait(&tfull[buf], (n >> 1) & 1, &g_int8_error)) break;
            __syncwarp();
            tc::fence_after();
            if (A.splits > 1) {  // this split's sums, for the first CTA of the cluster (one tile per cluster)
                int *part = (int *)smem + (q4 * 32 + lane) * (BN + 1);
                for (int c = 0; c < BN; c += 16) {
                    int v[16];
                    tc::tmem_ld16(tmem + lanes + (uint32_t)(buf * BN + c), v);
#pragma unroll
                    for (int i = 0; i < 16; i++) part[c + i] = v[i];
                }
                break;
            }
            const int64_t p = (int64_t)tp * 128 + q4 * 32 + lane;
            const float sp = SWAP ? (p < A.channels ? A.sb[p] : 0.0f) : (p < A.tokens ? A.sa[p] : 0.0f);
            const float bp = SWAP && A.bias && p < A.channels ? A.bias[p] : 0.0f;
#pragma unroll 1
            for (int c = 0; c < BN; c += 16) {
                int v[16];
                __syncwarp();
                tc::tmem_ld16(tmem + lanes + (uint32_t)(buf * BN + c), v);
                const int64_t q0 = (int64_t)tq * BN + c;
                if constexpr (SWAP) {  // a lane is a channel: 32 neighbours of one token's row per store
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        if (q0 + i < A.tokens && p < A.channels)
                            out[(q0 + i) * A.ldo + p] = from_f<T>(result(v[i], A.sa[q0 + i], sp, A.bias, bp));
                } else {
                    float y[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int64_t q = q0 + i < A.channels ? q0 + i : A.channels - 1;
                        y[i] = result(v[i], sp, A.sb[q], A.bias, A.bias ? A.bias[q] : 0.0f);
                    }
                    if (vec && q0 + 16 <= A.channels) {
                        if (p < A.tokens) {
                            alignas(16) T w[16];
#pragma unroll
                            for (int i = 0; i < 16; i++) w[i] = from_f<T>(y[i]);
#pragma unroll
                            for (int i = 0; i < (int)sizeof(w) / 16; i++)
                                ((uint4 *)(out + p * A.ldo + q0))[i] = ((const uint4 *)w)[i];
                        }
                    } else {  // turned in shared memory: 16 neighbours of each of two rows per store
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 16; i++) turn[lane * 33 + i] = y[i];
                        __syncwarp();
#pragma unroll
                        for (int r = 0; r < 32; r += 2) {
                            const int rr = r + (lane >> 4);
                            const int64_t row = (int64_t)tp * 128 + q4 * 32 + rr, q = q0 + (lane & 15);
                            if (row < A.tokens && q < A.channels) out[row * A.ldo + q] = from_f<T>(turn[rr * 33 + (lane & 15)]);
                        }
                    }
                }
            }
            tc::fence_before();
            tc::mb_arrive(&tfree[buf]);
        }
    }
    __syncwarp();
    if (A.splits > 1) {
        // all sums are in place (the stages' loads have all been read by then)
        cluster_sync();
        if (split == 0) {
            int tp, tq;
            place(blockIdx.x, &tp, &tq);
            T *out = (T *)A.out;
            for (int i = threadIdx.x; i < 128 * BN; i += TC_THREADS) {
                // neighbouring threads hold neighbouring channels
                const int pr = SWAP ? i & 127 : i / BN, qc = SWAP ? i >> 7 : i % BN;
                int sum = ((const int *)smem)[pr * (BN + 1) + qc];
                for (int r = 1; r < A.splits; r++) sum += ((const int *)cluster_map(smem, r))[pr * (BN + 1) + qc];
                const int64_t p = (int64_t)tp * 128 + pr, q = (int64_t)tq * BN + qc;
                const int64_t token = SWAP ? q : p, ch = SWAP ? p : q;
                if (token < A.tokens && ch < A.channels)
                    out[token * A.ldo + ch] = from_f<T>(result(sum, A.sa[token], A.sb[ch], A.bias, A.bias ? A.bias[ch] : 0.0f));
            }
        }
        cluster_sync();  // the others' shared memory stays until it has been read
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (warp == 1) tc::tmem_free(tmem, TT::COLS);
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        cudaDriverEntryPointQueryResult q;
        void *f = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            f = nullptr;
        }
        return (PFN_cuTensorMapEncodeTiled_v12000)f;
    }();
    return fn;
}

// Rows of `inner` bytes at a pitch of ld, in boxes of 128 bytes x box_rows.
bool make_map(CUtensorMap *map, const int8_t *base, int64_t inner, int64_t rows, int64_t ld, int box_rows) {
    cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
    cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, step[2] = {1, 1};
    const auto fn = encode_fn();
    return fn && fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void *)base, dims, strides, box, step,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN, bool SWAP, typename T>
int launch_tc(const CUtensorMap &mp, const CUtensorMap &mq, const TcArgs &A, cudaStream_t s) {
    auto k = int8_tc_kernel<BN, SWAP, T>;
    static bool attr[64] = {false};
    const int dev = current_device();
    if (dev < 0 || dev >= 64 || !attr[dev]) {
        ZC_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, TcTile<BN>::SMEM));
        if (dev >= 0 && dev < 64) attr[dev] = true;
    }
    const int64_t tiles = (int64_t)A.tiles_p * A.tiles_q;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(A.splits > 1 || tiles < num_sms() ? tiles : num_sms()), 1, (unsigned)A.splits);
    cfg.blockDim = dim3(TC_THREADS);
    cfg.dynamicSmemBytes = TcTile<BN>::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute at[1] = {};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = (unsigned)A.splits;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    ZC_CUDA(cudaLaunchKernelEx(&cfg, k, mp, mq, A));
    count_launch();
    return ZPUCUDA_OK;
}

// The tensor-core product of m x n x k: *done says whether its operands allow it.
template <typename T>
int product_tc(const int8_t *a, int64_t lda, const float *sa, const int8_t *b, int64_t ldb, const float *sb,
               const float *bias, T *out, int64_t ldo, int64_t m, int64_t n, int64_t k, cudaStream_t s, bool *done) {
    *done = false;
    // a tensor map's rows: at most 2^31, its coordinates 32 bits
    if (!aligned_to(a, 16) || !aligned_to(b, 16) || lda % 16 || ldb % 16 || k == 0) return ZPUCUDA_OK;
    // few tokens: weights along the 128 rows, the tokens in the narrowest tile that holds them
    const bool swap = m <= 128;
    const int bn = !swap ? 256 : m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128;
    TcArgs A = {sa, sb, bias, out, ldo, m, n};
    const int64_t P = swap ? n : m, Q = swap ? m : n;
    A.tiles_p = (int)((P + 127) / 128);
    A.tiles_q = (int)((Q + bn - 1) / bn);
    A.group = 16;
    A.kt = (int)((k + 127) / 128);
    // split the inner axis while the tiles leave most SMs idle, with at least four slices left to each
    int64_t splits = 1;
    const int64_t tiles = (int64_t)A.tiles_p * A.tiles_q;
    while (bn <= 128 && splits < 8 && tiles * splits * 2 <= num_sms() && A.kt / (splits * 2) >= 4) splits *= 2;
    A.kt_split = (int)((A.kt + splits - 1) / splits);
    A.splits = (A.kt + A.kt_split - 1) / A.kt_split;  // no split without a slice
    CUtensorMap mp, mq;
    if (!make_map(&mp, swap ? b : a, k, P, swap ? ldb : lda, 128) || !make_map(&mq, swap ? a : b, k, Q, swap ? lda : ldb, bn))
        return ZPUCUDA_OK;
    *done = true;
    if (!swap) return launch_tc<256, false, T>(mp, mq, A, s);
    if (bn == 16) return launch_tc<16, true, T>(mp, mq, A, s);
    if (bn == 32) return launch_tc<32, true, T>(mp, mq, A, s);
    if (bn == 64) return launch_tc<64, true, T>(mp, mq, A, s);
    return launch_tc<128, true, T>(mp, mq, A, s);
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
    bool done = false;
    ZC_HEAD_TYPE(dtype, T, ZC_TRY(product_tc<T>(a, lda, sa, b, ldb, sb, bias, (T *)out, ldo, m, n, k, s, &done)));
    if (done) return ZPUCUDA_OK;
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
