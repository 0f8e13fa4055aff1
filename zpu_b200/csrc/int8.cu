// The linear layer in 8-bit integers: rows quantised with one scale each,
//   scale = max |x| / 127,  q = round-half-to-even(x / scale)
// (a row of zeros keeps scale 0; a row with a NaN or an infinity gets scale
// NaN and q = 0, so only its own outputs become NaN), and the product
//   y[m, n] = (sum over k of a[m, k] * b[n, k]) * sa[m] * sb[n] + bias[n]
// whose sum is exact in 32-bit integers.
#include <string.h>

#include "head.cuh"
#include "tcgen05.cuh"
#include "waits.cuh"

namespace zc {

static __device__ unsigned int g_int8_error;

static std::atomic<bool> g_int8_waits{false};  // a kernel with waits has been launched

int int8_device_error(unsigned int *e) {
    if (!g_int8_waits.load(std::memory_order_relaxed)) return ZPUCUDA_OK;
    ZC_CUDA(cudaMemcpyFromSymbol(e, g_int8_error, sizeof *e));
    return ZPUCUDA_OK;
}

namespace {

constexpr int NT = 256;
// 131071 * 128 * 128 < 2^31: no sum of that many products leaves 32 bits.
constexpr int64_t kMaxInner = 131071;

// How long the warps that take finished sums (or arrived weights) wait for them, in tries, and where they tell of a wait that
// ran out (null: the library's own word).  Other waits, of copies and products in flight among them, keep the usual limit.
struct Patience {
    uint32_t limit = tc::kSpin;
    unsigned *err = nullptr;
    __device__ __forceinline__ unsigned *word() const { return err ? err : &g_int8_error; }
};

// One result from its sum, rounded alike on every path.
__device__ __forceinline__ float result(int sum, float sa, float sb, const float *bias, float b) {
    const float v = __fmul_rn(__fmul_rn((float)sum, sa), sb);
    return bias ? __fadd_rn(v, b) : v;
}

// rint(x / s) of n values as bytes, s > 0 and r = 1 / s rounded.  Adding 1.5 * 2^23
// rounds to a whole number (half to even) and leaves it in the low bits.  x * r is
// off by less than 127 * 2^-22 from x / s, so only a product that close to a tie
// needs the division (about one value in 10^4).
template <int N, typename T>
__device__ __forceinline__ void quantize_n(const T (&x)[N], float s, float r, int8_t (&q)[N]) {
    constexpr float magic = 12582912.0f;
    bool near = false;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float t = __fmul_rn(to_f(x[i]), r), u = __fadd_rn(t, magic);
        near |= fabsf(__fsub_rn(t, __fsub_rn(u, magic))) > 0.4999f;
        q[i] = (int8_t)__float_as_int(u);
    }
    if (near)
#pragma unroll
        for (int i = 0; i < N; i++) q[i] = (int8_t)__float_as_int(__fadd_rn(to_f(x[i]) / s, magic));
}

// The same for a piece of a row, two values an instruction.
template <typename T>
__device__ __forceinline__ void quantize_piece(const uint4 &x, float s, float r, int8_t (&q)[kPiece<T>]) {
    constexpr int N = kPiece<T>;
    const f32x2 magic = make2(12582912.0f), back = make2(-12582912.0f), minus = make2(-1.0f);
    f32x2 v[N / 2];
    unpack2<T>(x, v);
    float off = 0.0f;
    uint32_t b[N];
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
        const f32x2 t = mul2(v[i], make2(r)), u = add2(t, magic), d = fma2(add2(u, back), minus, t);
        off = fmaxf(off, fmaxf(fabsf(lo2(d)), fabsf(hi2(d))));
        b[2 * i] = __float_as_uint(lo2(u));
        b[2 * i + 1] = __float_as_uint(hi2(u));
    }
    if (off > 0.4999f)
#pragma unroll
        for (int i = 0; i < N; i++)
            b[i] = __float_as_uint(__fadd_rn((i & 1 ? hi2(v[i / 2]) : lo2(v[i / 2])) / s, 12582912.0f));
    uint32_t w[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; i++)
        w[i] = __byte_perm(__byte_perm(b[4 * i], b[4 * i + 1], 0x0040), __byte_perm(b[4 * i + 2], b[4 * i + 3], 0x0040), 0x5410);
    memcpy(q, w, N);
}
// The largest magnitude of a piece and m; NaN if there is one.
template <typename T>
__device__ __forceinline__ float largest_nan(const uint4 &x, float m) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    if constexpr (sizeof(T) == 2) {
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        T2 h[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t a = w[i] & 0x7fff7fffu;
            memcpy(&h[i], &a, 4);
        }
        const T2 t = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
        return max_nan(m, max_nan(to_f(t.x), to_f(t.y)));
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) m = max_nan(m, fabsf(__uint_as_float(w[i])));
        return m;
    }
}

// The same by its definition, for any scale (0 and NaN give 0).
__device__ __forceinline__ int8_t slow_quantized(float x, float s) {
    return s > 0.0f ? (int8_t)(int)fminf(fmaxf(rintf(x / s), -127.0f), 127.0f) : (int8_t)0;
}

// TPR threads hold a row in registers, V elements at a time (V > 1: 16-byte
// loads), NV times each; rows that this does not hold are read twice (NV = 0).
// One pass over HBM bounds it: 4096 x 8192 bf16 (100 MB moved) takes 25.5 us, 3.9
// TB/s; of values by themselves, not in pairs, 27.9 us.
template <typename T, int V, int TPR, int NV>
__global__ void __launch_bounds__(TPR < NT ? NT : TPR)
    quantize_kernel(const T *x, int64_t ldx, int8_t *q, int64_t ldq, float *scale, int64_t rows, int64_t cols) {
    constexpr int BLOCK = TPR < NT ? NT : TPR;
    __shared__ float sm[BLOCK / 32];
    struct alignas(V * sizeof(T)) Vec {
        T e[V];
    };
    struct alignas(V) Out {
        int8_t e[V];
    };
    const int64_t row = (int64_t)blockIdx.x * (BLOCK / TPR) + threadIdx.x / TPR;
    const int t = threadIdx.x % TPR;
    const bool in = row < rows;
    const T *xr = x + (in ? row : 0) * ldx;
    const int64_t n = cols / V, rest = n * V;  // whole vectors; the last cols % V elements are thread 0's
    Vec v[NV ? NV : 1];
    float m = 0.0f;
    auto widest = [&](const Vec &w) {
        if constexpr (V > 1) return largest_nan<T>(*(const uint4 *)&w, m);
        else return max_nan(m, fabsf(to_f(w.e[0])));
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; j++)
            if (in && t + j * TPR < n) v[j] = ((const Vec *)xr)[t + j * TPR];
#pragma unroll
        for (int j = 0; j < NV; j++)
            if (in && t + j * TPR < n) m = widest(v[j]);
    } else if (in) {
        for (int64_t i = t; i < n; i += TPR) m = widest(((const Vec *)xr)[i]);
    }
    if (V > 1 && in && t == 0)
        for (int64_t c = rest; c < cols; c++) m = max_nan(m, fabsf(to_f(xr[c])));
    m = warp_max_nan(m);
    if (TPR > 32) {
        if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = m;
        __syncthreads();
        const int w0 = threadIdx.x / TPR * (TPR / 32);
        m = sm[w0];
#pragma unroll
        for (int w = 1; w < TPR / 32; w++) m = max_nan(m, sm[w0 + w]);
    }
    if (!in) return;
    const float s = isfinite(m) ? m / 127.0f : NAN, r = 1.0f / s;
    const bool ok = s > 0.0f && isfinite(r);  // r overflows for a scale below 2^-128: divide
    int8_t *qr = q + row * ldq;
    auto put = [&](const Vec &w, int64_t i) {
        Out o;
        if (ok) {
            if constexpr (V > 1) quantize_piece<T>(*(const uint4 *)&w, s, r, o.e);
            else quantize_n(w.e, s, r, o.e);
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) o.e[e] = slow_quantized(to_f(w.e[e]), s);
        }
        ((Out *)qr)[i] = o;
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; j++)
            if (t + j * TPR < n) put(v[j], t + j * TPR);
    } else {
        for (int64_t i = t; i < n; i += TPR) put(((const Vec *)xr)[i], i);
    }
    if (t == 0) {
        if (V > 1)
            for (int64_t c = rest; c < cols; c++) qr[c] = slow_quantized(to_f(xr[c]), s);
        scale[row] = s;
    }
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

// The product of one or two tokens: the weights' bytes are all that counts, so
// they are streamed once, by bulk copies into shared memory: 16 warps with a ring
// of two 4 KiB slots each keep 128 KiB an SM in flight, and the first of them are
// on their way before the tokens are even read (loads into registers: 18.5 us
// where this takes 15.1, 16384 x 4096).  X is int8 (with its scales), or
// one of the head's types, which each block quantises for itself: one launch
// for a token's whole linear layer, 16.0 us from bf16 or 4.2 TB/s of weights.  A unit is a slot's worth: several short
// rows, or a piece of a long one; a block's units are dealt out evenly to its
// warps, and what a warp has of a channel goes to the block's whole-number sums.
struct VecArgs {
    const int8_t *w;
    const float *sx, *sw, *bias;
    int64_t ldx, ldw, ldo, n;
    int m, k;  // tokens, values
    int per, seg, segs, rows;  // VecUnits
    Patience wait;
};

template <int M, typename X, typename T>
__global__ void __launch_bounds__(GV_WARPS * 32, 1) int8_vec_kernel(const X *x, T *out, const VecArgs A) {
    extern __shared__ __align__(128) uint8_t vec_smem[];
    __shared__ int sums[GV_CHANNELS * M];
    __shared__ float red[M][GV_WARPS], scale[M];
    __shared__ uint64_t full[GV_WARPS][GV_SLOTS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, k = A.k;
    uint8_t *ring = vec_smem + warp * (GV_SLOTS * GV_SLOT);
    int8_t *xs = (int8_t *)vec_smem + GV_RING;
    const int pitch = vec_pitch(k);  // of the tokens' rows, zeros past k
    if (lane == 0) {
        for (int i = 0; i < GV_SLOTS; i++) tc::mb_init(&full[warp][i], 1);
        tc::mb_init_fence();
    }
    __syncwarp();

    bool first = true, ok = true;
    int issued = 0, used = 0;  // this warp's units, over all rounds
    for (int64_t c0 = (int64_t)blockIdx.x * A.per; c0 < A.n; c0 += (int64_t)gridDim.x * A.per) {
        const int nch = (int)(A.n - c0 < A.per ? A.n - c0 : A.per);
        const int units = (nch + A.rows - 1) / A.rows * A.segs;
        const int u0 = (int)((int64_t)units * warp / GV_WARPS), u1 = (int)((int64_t)units * (warp + 1) / GV_WARPS);
        int next = u0;
        auto issue = [&]() {  // lane 0: unit `next` into its slot
            const int slot = issued % GV_SLOTS, piece = next % A.segs, ch = next / A.segs * A.rows;
            const int rows = min(A.rows, nch - ch), at = piece * A.seg, rest = k - at;
            uint8_t *dst = ring + slot * GV_SLOT;
            const int8_t *src = A.w + (c0 + ch) * A.ldw + at;
            // 16 bytes that begin inside a row end inside its pitch (a multiple of 16), and what lies past k meets
            // zeros; the last row may end with the memory, so its last bytes come one by one
            const int size = min(A.seg, (rest + 15) & ~15);
            const bool last = c0 + ch + rows == A.n && (rest & 15) && rest < A.seg;
            const int lsize = last ? rest & ~15 : size;
            if (last)
                for (int b = lsize; b < rest; b++) dst[(rows - 1) * A.seg + b] = (uint8_t)src[(rows - 1) * A.ldw + b];
            tc::mb_expect_tx(&full[warp][slot], (uint32_t)(size * (rows - 1) + lsize));
            for (int r = 0; r < rows; r++) {
                const int n = r == rows - 1 ? lsize : size;
                if (n)
                    asm volatile(
                        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                            tc::su32(dst + r * A.seg)),
                        "l"(src + r * A.ldw), "r"(n), "r"(tc::su32(&full[warp][slot]))
                        : "memory");
            }
            next++;
            issued++;
        };
        if (lane == 0)
            while (ok && next < u1 && issued - used < GV_SLOTS) issue();
        for (int i = threadIdx.x; i < M * nch; i += GV_WARPS * 32) sums[i] = 0;
        if (first) {  // the tokens, while the first weights are on their way
            first = false;
            for (int i = threadIdx.x; i < M * pitch / 16; i += GV_WARPS * 32) ((uint4 *)xs)[i] = make_uint4(0, 0, 0, 0);
            if constexpr (sizeof(X) == 1) {
                __syncthreads();
                for (int r = 0; r < A.m; r++) {
                    const int n = ((uintptr_t)x & 15) == 0 && A.ldx % 16 == 0 ? k / 16 : 0;
                    for (int i = threadIdx.x; i < n; i += GV_WARPS * 32)
                        ((uint4 *)(xs + r * pitch))[i] = ((const uint4 *)(x + r * A.ldx))[i];
                    for (int c = n * 16 + threadIdx.x; c < k; c += GV_WARPS * 32) xs[r * pitch + c] = x[r * A.ldx + c];
                }
                if (threadIdx.x < A.m) scale[threadIdx.x] = A.sx[threadIdx.x];
            } else {
                constexpr int V = 16 / sizeof(X);
                struct alignas(16) Vec {
                    X e[V];
                };
                struct alignas(V) Out {
                    int8_t e[V];
                };
                const int n = ((uintptr_t)x & 15) == 0 && A.ldx % V == 0 ? k / V : 0;  // whole vectors
#pragma unroll
                for (int r = 0; r < M; r++) {
                    float top = 0.0f;
                    if (r < A.m) {
                        const X *xr = x + r * A.ldx;
                        for (int i = threadIdx.x; i < n; i += GV_WARPS * 32) {
                            const Vec v = ((const Vec *)xr)[i];
#pragma unroll
                            for (int e = 0; e < V; e++) top = max_nan(top, fabsf(to_f(v.e[e])));
                        }
                        for (int c = n * V + threadIdx.x; c < k; c += GV_WARPS * 32) top = max_nan(top, fabsf(to_f(xr[c])));
                    }
                    top = warp_max_nan(top);
                    if (lane == 0) red[r][warp] = top;
                }
                __syncthreads();
#pragma unroll
                for (int r = 0; r < M; r++) {
                    if (r >= A.m) break;
                    const X *xr = x + r * A.ldx;
                    const float t = warp_max_nan(red[r][lane % GV_WARPS]);
                    const float s = isfinite(t) ? t / 127.0f : NAN, inv = 1.0f / s;
                    const bool quick = s > 0.0f && isfinite(inv);
                    for (int i = threadIdx.x; i < n; i += GV_WARPS * 32) {
                        const Vec v = ((const Vec *)xr)[i];
                        Out o;
                        if (quick) {
                            quantize_n(v.e, s, inv, o.e);
                        } else {
#pragma unroll
                            for (int e = 0; e < V; e++) o.e[e] = slow_quantized(to_f(v.e[e]), s);
                        }
                        ((Out *)(xs + r * pitch))[i] = o;
                    }
                    for (int c = n * V + threadIdx.x; c < k; c += GV_WARPS * 32) xs[r * pitch + c] = slow_quantized(to_f(xr[c]), s);
                    if (threadIdx.x == 0) scale[r] = s;
                }
            }
        }
        __syncthreads();

        int acc[M] = {};
        for (int u = u0; u < u1; u++) {
            const int slot = used % GV_SLOTS, piece = u % A.segs, ch = u / A.segs * A.rows;
            if (!__all_sync(0xffffffffu, ok && tc::mb_wait(&full[warp][slot], (used / GV_SLOTS) & 1, A.wait.word(), A.wait.limit))) {
                ok = false;
                break;
            }
            const uint8_t *src = ring + slot * GV_SLOT;
            const int rows = min(A.rows, nch - ch), size = min(A.seg, k - piece * A.seg);
            const int8_t *xp = xs + piece * A.seg + lane * 16;
            auto step = [&](int (&sum)[M], const uint8_t *row, const int4 (&y)[M]) {
                const int4 v = *(const int4 *)(row + lane * 16);
#pragma unroll
                for (int t = 0; t < M; t++) {
                    sum[t] = __dp4a(v.x, y[t].x, sum[t]);
                    sum[t] = __dp4a(v.y, y[t].y, sum[t]);
                    sum[t] = __dp4a(v.z, y[t].z, sum[t]);
                    sum[t] = __dp4a(v.w, y[t].w, sum[t]);
                }
            };
            auto token = [&](int4 (&y)[M], int at) {
#pragma unroll
                for (int t = 0; t < M; t++) y[t] = *(const int4 *)(xp + t * pitch + at);
            };
            auto flush = [&](int (&sum)[M], int c) {
#pragma unroll
                for (int t = 0; t < M; t++) {
                    const int s = __reduce_add_sync(0xffffffffu, sum[t]);
                    if (lane == 0) atomicAdd(&sums[c * M + t], s);
                    sum[t] = 0;
                }
            };
            int4 y[M];
            if (A.rows == 1) {  // a piece of one row, in steps that do not wait for one another's loads
                int at = 0;
                for (; at + 2048 <= size; at += 2048)
#pragma unroll
                    for (int i = 0; i < 2048; i += 512) {
                        token(y, at + i);
                        step(acc, src + at + i, y);
                    }
                for (; at < size; at += 512)
                    if (at + lane * 16 < size) {
                        token(y, at);
                        step(acc, src + at, y);
                    }
                __syncwarp();
                if (piece == A.segs - 1 || u == u1 - 1) flush(acc, ch);  // all that this warp has of the channel
            } else {  // four short rows at a time (what the last row gives again is left out)
                for (int r = 0; r < rows; r += 4) {
                    int sum[4][M] = {};
                    const uint8_t *from[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) from[i] = src + vec_row(r + i, rows) * A.seg;
                    for (int at = 0; at < size; at += 512)
                        if (at + lane * 16 < size) {
                            token(y, at);
#pragma unroll
                            for (int i = 0; i < 4; i++) step(sum[i], from[i] + at, y);
                        }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (r + i < rows) flush(sum[i], ch + r + i);
                }
            }
            __syncwarp();  // the slot has been read
            used++;
            if (lane == 0 && next < u1) issue();
            issued = __shfl_sync(0xffffffffu, issued, 0);
            next = __shfl_sync(0xffffffffu, next, 0);
        }
        const bool lost = __syncthreads_or(!ok);  // the sums lack what a warp has given up on: NaN
        for (int i = threadIdx.x; i < nch * A.m; i += GV_WARPS * 32) {
            const int c = i % nch, r = i / nch;
            out[r * A.ldo + c0 + c] = from_f<T>(
                result(sums[c * M + r], lost ? NAN : scale[r], A.sw[c0 + c], A.bias, A.bias ? A.bias[c0 + c] : 0.0f));
        }
        __syncthreads();  // the sums have been read
    }
    if (!ok && lane == 0)  // give up only once the copies in flight have landed
        for (int i = used; i < issued; i++) tc::mb_wait(&full[warp][i % GV_SLOTS], (i / GV_SLOTS) & 1, A.wait.word());
}

// Whether the kernel above takes m tokens of k values: they fit its shared memory.
// (Four tokens with 16384 x 4096 weights took 25 us, on the tensor cores 18.)
bool takes_vec(const int8_t *w, int64_t ldw, int64_t m, int64_t k) {
    return m >= 1 && m <= 2 && k > 0 && aligned_to(w, 16) && ldw % 16 == 0 && m * vec_pitch((int)k) <= GV_X;
}

template <int M, typename X, typename T>
int launch_vec(const X *x, T *out, VecArgs A, cudaStream_t s) {
    auto f = int8_vec_kernel<M, X, T>;
    static bool attr[64] = {false};
    const int dev = current_device();
    if (dev < 0 || dev >= 64 || !attr[dev]) {
        ZC_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, GV_RING + GV_X));
        if (dev >= 0 && dev < 64) attr[dev] = true;
    }
    const VecUnits U = vec_units(A.n, A.k, num_sms());
    A.per = U.per;
    A.seg = U.seg;
    A.segs = U.segs;
    A.rows = U.rows;
    const int64_t blocks = (A.n + U.per - 1) / U.per;
    const size_t smem = vec_smem(M, A.k);
    f<<<(unsigned)(blocks < num_sms() ? blocks : num_sms()), GV_WARPS * 32, smem, s>>>(x, out, A);
    ZC_LAUNCHED("int8_vec_kernel");
    return ZPUCUDA_OK;
}
template <typename X, typename T>
int product_vec(const X *x, int64_t ldx, const float *sx, const int8_t *w, int64_t ldw, const float *sw, const float *bias,
                T *out, int64_t ldo, int64_t m, int64_t n, int64_t k, const Patience &wait, cudaStream_t s) {
    VecArgs A = {w, sx, sw, bias, ldx, ldw, ldo, n, (int)m, (int)k};
    A.wait = wait;
    return m == 1 ? launch_vec<1>(x, out, A, s) : launch_vec<2>(x, out, A, s);
}

// A product on the tensor cores: D[p, q] = sum over k of P[p, k] * Q[q, k] in
// tiles of 128 x BN, for operands that a tensor map can describe (addresses
// and row pitches multiples of 16 bytes).  P is a and Q is b, or (SWAP) P is b
// and Q is a: with few tokens the weights fill the 128 rows and a narrow tile
// holds the tokens, so no multiplication is spent on rows that are not there.
//
// One CTA per SM walks tiles; warp 0 loads 128-byte slices of both operands by
// TMA into a ring of stages, one lane of warp 1 issues tcgen05.mma (kind::i8,
// exact 32-bit sums in TMEM), warps 2-9 turn a finished tile into the result
// while the next one is summed into the other TMEM buffer.  With few tiles the
// inner axis is split over a cluster, whose CTAs add up each other's sums through
// shared memory (whole numbers: the split does not change the result).
//
// The tensor cores bound a large product: 4096 x 8192 x 8192 takes 171 to 192 us, 2.9e15
// operations a second or more, at the power limit's clock; 128 x 256 tiles read half as
// much from L2 a product as 128 x 128 ones.  Small ones are bound by the way from
// the first load to the last store: 333 x 4099 x 1001 takes 9 us.
constexpr int TC_THREADS = 320;  // producer, issuer, eight storing warps
constexpr int TC_STAGE_A = 128 * 128;
template <int BN>
struct TcTile {
    static constexpr int STAGE = TC_STAGE_A + BN * 128;
    static constexpr int STAGES = BN == 256 ? 4 : BN == 128 ? 6 : 8;
    static constexpr int COLS = 2 * BN < 32 ? 32 : 2 * BN;  // two sums in TMEM
    static constexpr int PART = BN * 132 * 4;               // a split's sums, one Q row after another
    static constexpr int TURN = 8 * 32 * 64;                // 32 rows of 64 bytes of each storing warp
    static constexpr int SMEM = STAGES * STAGE + TURN + 1024;
    static_assert(SMEM + 16 * BN + 512 <= 227 * 1024 && (BN == 256 || PART <= STAGES * STAGE), "shared memory");
};

struct TcArgs {
    const float *sa, *sb, *bias;  // by token, by channel
    void *out;
    int64_t ldo, tokens, channels;
    int tiles_p, tiles_q, group;  // tiles along P and Q; P tiles per raster group
    int kt, kt_split, splits;     // 128-byte slices, slices of a split
    Patience wait;
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
    __shared__ uint64_t full[TT::STAGES], empty[TT::STAGES], tfull[2], tfree[2], drained;
    __shared__ uint32_t tmem_base, gave_up;  // a split's sums are not in place
    __shared__ float sq[2][BN], bq[2][BN];  // the Q side's scales and biases, of this tile and the next
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
            tc::mb_init(&tfree[b], 256);
        }
        tc::mb_init(&drained, 1);
        gave_up = 0;
        tc::mb_init_fence();
    }
    if (warp == 1) tc::tmem_alloc(&tmem_base, TT::COLS);
    asm volatile("griddepcontrol.wait;" ::: "memory");  // where the quantising kernel may still run
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
                    if (j >= TT::STAGES && !tc::mb_wait(&empty[s], ((j / TT::STAGES) - 1) & 1, A.wait.word())) {
                        ok = false;
                        break;
                    }
                    uint8_t *st = smem + s * TT::STAGE;
                    tc::mb_expect_tx(&full[s], TT::STAGE);
                    tc::tma_load_2d(st, &mp, k * 128, tp * 128, &full[s]);
                    tc::tma_load_2d(st + TC_STAGE_A, &mq, k * 128, tq * BN, &full[s]);
                }
            }
            // the block ends only once the copies in flight have landed, also where nobody waits for them any more
            for (int i = max(0, j - TT::STAGES); i < j; i++)
                tc::mb_wait(&full[i % TT::STAGES], (i / TT::STAGES) & 1, A.wait.word());
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t ID = tc::idesc_s8(128, BN);
            int j = 0, n = 0;
            bool ok = true;
            for (int t = blockIdx.x; t < ntiles && ok; t += gridDim.x, n++) {
                const int buf = n & 1;
                if (n >= 2 && !tc::mb_wait(&tfree[buf], ((n >> 1) - 1) & 1, A.wait.word())) {
                    ok = false;
                    break;
                }
                tc::fence_after();
                for (int k = k0; k < k1; k++, j++) {
                    const int s = j % TT::STAGES;
                    if (!tc::mb_wait(&full[s], (j / TT::STAGES) & 1, A.wait.word())) {
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
            // nor while products are on their way to TMEM (those of finished tiles are waited for by the storing warps, in time or
            // not)
            if (!ok) {
                tc::mma_commit(&drained);
                tc::mb_wait(&drained, 0, A.wait.word());
            }
        }
    } else {
        // warp w reads the quarter w % 4 of the TMEM lanes, and one half of the columns
        constexpr int HALF = BN >= 32 ? BN / 2 : BN;
        const int q4 = warp & 3, half = (warp - 2) >> 2;
        const uint32_t lanes = (uint32_t)(q4 * 32) << 16;
        const bool idle = half * HALF >= BN;
        T *out = (T *)A.out;
        uint8_t *turn = smem + TT::STAGES * TT::STAGE + (warp - 2) * 2048;
        const bool vec = ((uintptr_t)out & 15) == 0 && (A.ldo * (int64_t)sizeof(T)) % 16 == 0;
        int n = 0;
        bool good = true, coming = true;  // the warp's: no wait has run out; nor one at the usual limit after that
        for (int t = blockIdx.x; t < ntiles; t += gridDim.x, n++) {
            int tp, tq;
            place(t, &tp, &tq);
            const int buf = n & 1;
            const int64_t p = (int64_t)tp * 128 + q4 * 32 + lane;
            float sp = 0.0f, bp = 0.0f;
            if (A.splits == 1) {  // the scales, while the sums are being made
                for (int i = threadIdx.x - 64; i < BN; i += 256) {
                    const int64_t q = (int64_t)tq * BN + i;
                    const bool in = q < (SWAP ? A.tokens : A.channels);
                    sq[buf][i] = in ? (SWAP ? A.sa[q] : A.sb[q]) : 0.0f;
                    if (!SWAP) bq[buf][i] = in && A.bias ? A.bias[q] : 0.0f;
                }
                if (p < (SWAP ? A.channels : A.tokens)) sp = SWAP ? A.sb[p] : A.sa[p];
                if (SWAP && A.bias && p < A.channels) bp = A.bias[p];
                asm volatile("bar.sync 1, 256;" ::: "memory");
            }
            good = __all_sync(0xffffffffu, good && tc::mb_wait(&tfull[buf], (n >> 1) & 1, A.wait.word(), A.wait.limit));
            if (!good) {
                // NaN from here on, but the barriers of the tiles to come are met (another warp's wait may have been in time),
                // at the pace of the sums as long as they come: the issuing warp counts on never being passed.
                coming = __all_sync(0xffffffffu, coming && tc::mb_wait(&tfull[buf], (n >> 1) & 1, A.wait.word()));
                sp = NAN;
            }
            tc::fence_after();
            auto sums = [&](int c, int (&v)[16]) {
                if (good) tc::tmem_ld16(tmem + lanes + (uint32_t)(buf * BN + c), v);
                else memset(v, 0, sizeof v);
            };
            if (A.splits > 1) {  // this split's sums, for the whole cluster (one tile per cluster)
                if (!good) gave_up = 1;
                int *part = (int *)smem + q4 * 32 + lane;
                for (int c = half * HALF; !idle && c < half * HALF + HALF; c += 16) {
                    int v[16];
                    sums(c, v);
#pragma unroll
                    for (int i = 0; i < 16; i++) part[(c + i) * 132] = v[i];
                }
                break;
            }
            if constexpr (SWAP) {  // a lane is a channel: 32 neighbours of one token's row per store
                for (int c = half * HALF; !idle && c < half * HALF + HALF; c += 16) {
                    int v[16];
                    __syncwarp();
                    sums(c, v);
                    const int64_t q0 = (int64_t)tq * BN + c;
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        if (q0 + i < A.tokens && p < A.channels)
                            out[(q0 + i) * A.ldo + p] = from_f<T>(result(v[i], sq[buf][c + i], sp, A.bias, bp));
                }
            } else {
                // 32 rows of 64 bytes turned in shared memory (16-byte piece u of row r at
                // u ^ (r / 2 % 4)), so that a store writes 64 bytes of each of eight rows
                constexpr int W = 64 / sizeof(T), E = 16 / sizeof(T);
#pragma unroll 1
                for (int c = half * HALF; c < half * HALF + HALF; c += W) {
                    __syncwarp();
#pragma unroll
                    for (int h = 0; h < W; h += 16) {
                        int v[16];
                        sums(c + h, v);
                        alignas(16) T w[16];
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            w[i] = from_f<T>(result(v[i], sp, sq[buf][c + h + i], A.bias, bq[buf][c + h + i]));
#pragma unroll
                        for (int u = 0; u < 16 / E; u++)
                            *(uint4 *)(turn + lane * 64 + (((h / E + u) ^ (lane >> 1 & 3)) * 16)) = ((const uint4 *)w)[u];
                    }
                    __syncwarp();
                    const int64_t q0 = (int64_t)tq * BN + c, p0 = (int64_t)tp * 128 + q4 * 32;
                    if (vec && q0 + W <= A.channels) {
#pragma unroll
                        for (int r = 0; r < 32; r += 8) {
                            const int rr = r + (lane >> 2), u = lane & 3;
                            if (p0 + rr < A.tokens)
                                *(uint4 *)(out + (p0 + rr) * A.ldo + q0 + u * E) =
                                    *(const uint4 *)(turn + rr * 64 + ((u ^ (rr >> 1 & 3)) * 16));
                        }
                    } else {
                        const int rows = (int)(A.tokens - p0 < 32 ? A.tokens - p0 : 32);
                        constexpr int R = 32 / W;  // rows of a store
                        const int j = lane % W;
                        if (q0 + j < A.channels)
                            for (int r = lane / W; r < rows; r += R)
                                out[(p0 + r) * A.ldo + q0 + j] =
                                    *(const T *)(turn + r * 64 + (((j / E) ^ (r >> 1 & 3)) * 16) + (j % E) * sizeof(T));
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
        // each CTA adds up its share: four neighbouring channels of a token a thread
        int tp, tq;
        place(blockIdx.x, &tp, &tq);
        T *out = (T *)A.out;
        const int share = (BN + A.splits - 1) / A.splits, first = split * share, end = min(BN, first + share);
        for (int i = threadIdx.x; i < (end - first) * 32; i += TC_THREADS) {
            const int qc = first + (i >> 5), at = qc * 132 + (i & 31) * 4;
            const int64_t token = (int64_t)tq * BN + qc, ch = (int64_t)tp * 128 + (i & 31) * 4;
            if (token >= A.tokens || ch >= A.channels) continue;
            int4 sum = make_int4(0, 0, 0, 0);
            uint32_t lost = 0;
#pragma unroll 8
            for (int r = 0; r < A.splits; r++) {
                const int4 v = *(const int4 *)((const int *)cluster_map(smem, r) + at);
                sum.x += v.x;
                sum.y += v.y;
                sum.z += v.z;
                sum.w += v.w;
                lost |= *(const uint32_t *)cluster_map(&gave_up, r);
            }
            const int y[4] = {sum.x, sum.y, sum.z, sum.w};
            const float sa = lost ? NAN : A.sa[token];
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (ch + e < A.channels)
                    out[token * A.ldo + ch + e] = from_f<T>(result(y[e], sa, A.sb[ch + e], A.bias, A.bias ? A.bias[ch + e] : 0.0f));
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
int launch_tc(const CUtensorMap &mp, const CUtensorMap &mq, const TcArgs &A, bool follows, cudaStream_t s) {
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
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = (unsigned)A.splits;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = follows ? 2 : 1;
    ZC_CUDA(cudaLaunchKernelEx(&cfg, k, mp, mq, A));
    count_launch();
    return ZPUCUDA_OK;
}

// The tensor-core product of m x n x k: *done says whether its operands allow it.  follows: the kernel launched last on the
// stream made the left operand, and this one's beginning may overlap its end.
template <typename T>
int product_tc(const int8_t *a, int64_t lda, const float *sa, const int8_t *b, int64_t ldb, const float *sb,
               const float *bias, T *out, int64_t ldo, int64_t m, int64_t n, int64_t k, bool follows,
               const Patience &wait, cudaStream_t s, bool *done) {
    *done = false;
    // a tensor map's rows: at most 2^31, its coordinates 32 bits
    if (!aligned_to(a, 16) || !aligned_to(b, 16) || lda % 16 || ldb % 16 || k == 0) return ZPUCUDA_OK;
    // few tokens: weights along the 128 rows, the tokens in the narrowest tile that holds them; so too where
    // the tiles fill less than half of the SMs and the inner axis will be split
    const bool swap = m <= 128 || (m + 127) / 128 * ((n + 127) / 128) * 2 <= num_sms();
    // wide tiles read half as much per product (4096 x 8192 by 8192: 192 us, 297 with narrow ones); narrow ones where they fill
    // the SMs' last wave better by the count of waves, in which a wide one stands for two
    const auto waves = [&](int w) { return ((m + 127) / 128 * ((n + w - 1) / w) + num_sms() - 1) / num_sms(); };
    const int wide = 2 * waves(256) <= waves(128) ? 256 : 128;
    const int bn = !swap ? wide : m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128;
    TcArgs A = {sa, sb, bias, out, ldo, m, n};
    const int64_t P = swap ? n : m, Q = swap ? m : n;
    A.tiles_p = (int)((P + 127) / 128);
    A.tiles_q = (int)((Q + bn - 1) / bn);
    A.group = 16;
    A.wait = wait;
    A.kt = (int)((k + 127) / 128);
    // split the inner axis while the tiles leave most SMs idle, with at least four slices left to each (16 x 4096 by 1024: 6.7
    // us, with eight left 7.9; with two left 8 x 2048 by 512 takes 5.6 instead of 6.4, but 16 x 512 by 2048 6.0 instead of 5.4)
    int64_t splits = 1;
    const int64_t tiles = (int64_t)A.tiles_p * A.tiles_q;
    while (swap && splits < 8 && tiles * splits * 2 <= num_sms() && A.kt / (splits * 2) >= 4) splits *= 2;
    A.kt_split = (int)((A.kt + splits - 1) / splits);
    A.splits = (A.kt + A.kt_split - 1) / A.kt_split;  // no split without a slice
    CUtensorMap mp, mq;
    if (!make_map(&mp, swap ? b : a, k, P, swap ? ldb : lda, 128) || !make_map(&mq, swap ? a : b, k, Q, swap ? lda : ldb, bn))
        return ZPUCUDA_OK;
    *done = true;
    if (!swap) return bn == 256 ? launch_tc<256, false, T>(mp, mq, A, follows, s) : launch_tc<128, false, T>(mp, mq, A, follows, s);
    if (bn == 16) return launch_tc<16, true, T>(mp, mq, A, follows, s);
    if (bn == 32) return launch_tc<32, true, T>(mp, mq, A, follows, s);
    if (bn == 64) return launch_tc<64, true, T>(mp, mq, A, follows, s);
    return launch_tc<128, true, T>(mp, mq, A, follows, s);
}

template <typename T, int V>
int launch_quantize(const T *x, int64_t ldx, int8_t *q, int64_t ldq, float *scale, int64_t rows, int64_t cols,
                    cudaStream_t s) {
    constexpr int NV = V > 1 ? 4 : 16;
    const int64_t n = cols / V;
    auto go = [&](auto f, int tpr) {
        const int block = tpr < NT ? NT : tpr;
        f<<<(unsigned)((rows + block / tpr - 1) / (block / tpr)), block, 0, s>>>(x, ldx, q, ldq, scale, rows, cols);
    };
    // As few threads a row as hold it in registers (4096 x 2048 bf16 takes 10.3 us with 64, 13.7 with 256), but 256 where
    // there are few rows (64 x 4096 bf16: 2.5 us, with 128 3.2; 333 x 1001 3.0, with 64 4.0).
    const bool few = rows <= 4 * (int64_t)num_sms();
    if (n <= 32 * NV) go(quantize_kernel<T, V, 32, NV>, 32);
    else if (n <= 64 * NV && !few) go(quantize_kernel<T, V, 64, NV>, 64);
    else if (n <= 128 * NV && !few) go(quantize_kernel<T, V, 128, NV>, 128);
    else if (n <= 256 * NV) go(quantize_kernel<T, V, 256, NV>, 256);
    else if (n <= 512 * NV) go(quantize_kernel<T, V, 512, NV>, 512);
    else if (n <= 1024 * NV) go(quantize_kernel<T, V, 1024, NV>, 1024);
    else go(quantize_kernel<T, V, 1024, 0>, 1024);
    ZC_LAUNCHED("quantize_kernel");
    return ZPUCUDA_OK;
}

int quantize(int dtype, const void *x, int64_t ldx, int8_t *q, int64_t ldq, float *scale, int64_t rows, int64_t cols,
             cudaStream_t s) {
    if (rows == 0) return ZPUCUDA_OK;
    const int V = 16 / elem_bytes(dtype);
    const bool vec = aligned_to(x, 16) && ldx % V == 0 && aligned_to(q, V) && ldq % V == 0;
    ZC_HEAD_TYPE(dtype, T, {
        constexpr int W = 16 / sizeof(T);
        return vec ? launch_quantize<T, W>((const T *)x, ldx, q, ldq, scale, rows, cols, s)
                   : launch_quantize<T, 1>((const T *)x, ldx, q, ldq, scale, rows, cols, s);
    });
}

int product(const int8_t *a, int64_t lda, const float *sa, const int8_t *b, int64_t ldb, const float *sb,
            const float *bias, int dtype, void *out, int64_t ldo, int64_t m, int64_t n, int64_t k, bool follows,
            cudaStream_t s, const Patience &wait = Patience()) {
    if (m == 0 || n == 0) return ZPUCUDA_OK;
    g_int8_waits.store(true, std::memory_order_relaxed);
    if (takes_vec(b, ldb, m, k))
        ZC_HEAD_TYPE(dtype, T, return (product_vec<int8_t, T>(a, lda, sa, b, ldb, sb, bias, (T *)out, ldo, m, n, k, wait, s)));
    bool done = false;
    ZC_HEAD_TYPE(dtype, T, ZC_TRY(product_tc<T>(a, lda, sa, b, ldb, sb, bias, (T *)out, ldo, m, n, k, follows, wait, s, &done)));
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
    return check_vectors(who, 4, {{"b's scales", sb}, {"bias", bias}});
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
    ZC_TRY(check_vectors("int8_quantize", 4, {{"scale", d_scale}}));
    if (ldq < cols) return set_error(ZPUCUDA_ERR_INVALID_SHAPE, "int8_quantize: q: row pitch below the row's length");
    if (rows > 0 && ((cols > 0 && !d_q) || !d_scale))
        return set_error(ZPUCUDA_ERR_INVALID_ARGUMENT, "int8_quantize: q or scale: null pointer");
    return quantize(dtype, d_x, ldx, d_q, ldq, d_scale, rows, cols, resolve_stream(stream));
}

static int int8_matmul(const char *who, const int8_t *a, int64_t lda, const float *sa, const int8_t *b, int64_t ldb,
                       const float *sb, const float *bias, int dtype, void *out, int64_t ldo, int64_t m, int64_t n,
                       int64_t k, const Patience &wait, void *stream) {
    ZC_TRY(check_product(who, sb, b, ldb, bias, dtype, out, ldo, m, n, k));
    if (lda < k) return head_error(ZPUCUDA_ERR_INVALID_SHAPE, who, "a: row pitch below the row's length");
    ZC_TRY(check_vectors(who, 4, {{"a's scales", sa}}));
    if (m > 0 && ((k > 0 && !a) || !sa)) return head_error(ZPUCUDA_ERR_INVALID_ARGUMENT, who, "a or its scales: null pointer");
    return product(a, lda, sa, b, ldb, sb, bias, dtype, out, ldo, m, n, k, false, resolve_stream(stream), wait);
}

int zpucuda_int8_matmul(const int8_t *d_a, int64_t lda, const float *d_sa, const int8_t *d_b, int64_t ldb,
                        const float *d_sb, const float *d_bias, int dtype, void *d_out, int64_t ldo, int64_t m,
                        int64_t n, int64_t k, void *stream) {
    return int8_matmul("int8_matmul", d_a, lda, d_sa, d_b, ldb, d_sb, d_bias, dtype, d_out, ldo, m, n, k, Patience(), stream);
}

int zpucuda_debug_int8_matmul(const int8_t *d_a, int64_t lda, const float *d_sa, const int8_t *d_b, int64_t ldb,
                              const float *d_sb, const float *d_bias, int dtype, void *d_out, int64_t ldo, int64_t m,
                              int64_t n, int64_t k, uint32_t spin_limit, uint32_t *d_err, void *stream) {
    ZC_TRY(check_vectors("debug_int8_matmul", 4, {{"err", d_err}}));
    Patience wait;
    wait.limit = spin_limit;
    wait.err = d_err;
    return int8_matmul("debug_int8_matmul", d_a, lda, d_sa, d_b, ldb, d_sb, d_bias, dtype, d_out, ldo, m, n, k, wait, stream);
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
    // The one launch for one or two tokens has every block read x while others store y: where the two share memory, x is
    // quantised in a launch of its own, as it is for more tokens.
    const int64_t e = elem_bytes(dtype);
    const uintptr_t x0 = (uintptr_t)d_x, x1 = x0 + ((rows - 1) * ldx + inner) * e, y0 = (uintptr_t)d_y,
                    y1 = y0 + ((rows - 1) * ldy + cols) * e;
    const bool apart = x1 <= y0 || y1 <= x0;
    g_int8_waits.store(true, std::memory_order_relaxed);
    if (apart && takes_vec(d_w, ldw, rows, inner))
        ZC_HEAD_TYPE(dtype, T, return (product_vec<T, T>((const T *)d_x, ldx, nullptr, d_w, ldw, d_sw, d_bias, (T *)d_y,
                                                         ldy, rows, cols, inner, Patience(), s)));
    const int64_t ldq = (inner + 15) / 16 * 16;
    int8_t *q = (int8_t *)d_work;
    float *scale = (float *)(q + rows * ldq);
    ZC_TRY(quantize(dtype, d_x, ldx, q, ldq, scale, rows, inner, s));
    return product(q, ldq, scale, d_w, ldw, d_sw, d_bias, dtype, d_y, ldy, rows, cols, inner, true, s);
}

int64_t zpucuda_int8_linear_work(int64_t rows, int64_t inner) {
    if (rows < 0 || inner < 0) return 0;
    return rows * ((inner + 15) / 16 * 16) + rows * 4;
}

}  // extern "C"
