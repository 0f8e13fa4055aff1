// Distillation of a student's logits from a teacher's top logits, and its
// gradient.  Per row, with z = logits / T over the vocabulary and the K
// listed teacher logits u = teacher / T at indices i:
//   q = softmax(z),  p = softmax(u over the listed entries)
//   loss = weight * T^2 * sum over k of p_k * (log p_k - log q[i_k])
//   dlogits_v = c * (q_v - sum over {k: i_k = v} of p_k),  c = T * weight * dloss.
// A listed index of -1 is no entry; a row without an entry of weight (none
// listed, or all of them -inf), with weight 0 or (gradient) c = 0 gives 0
// and its logits are not read.  Any other index outside [0, vocab) makes its
// row NaN.
// HBM bounds it, with the exponential unit close behind (two exponentials an
// element where both loss and gradient are wanted).  A row is split over the
// blocks of a cluster: each reads its slice once for maximum and sum, the blocks
// exchange those, and the gradient reads the slice again, from L2, where it has
// stayed (slices are at most 64 KiB, so all that is in flight is a third of L2).
// Holding slices in shared memory instead was slower: every byte then occupies
// its place from the copy to the gradient, 13.7 us, and 192 KiB an SM do not
// cover that time at HBM's rate (2048 x 131072 bf16: 270 us, 230 us now, 4.7 TB/s;
// the loss alone 135 us, bound by its exponential: 4.0 TB/s).
// A slice is counted in aligned 16-byte granules of memory, so an odd vocabulary
// costs two partial granules a row and nothing else.
#include "head.cuh"
#include "tcgen05.cuh"
#include "waits.cuh"

namespace zc {

static __device__ unsigned int g_distill_error;

static std::atomic<bool> g_distill_waits{false};  // a kernel with waits has been launched

int distill_device_error(unsigned int *e) {
    if (!g_distill_waits.load(std::memory_order_relaxed)) return ZPUCUDA_OK;
    ZC_CUDA(cudaMemcpyFromSymbol(e, g_distill_error, sizeof *e));
    return ZPUCUDA_OK;
}

namespace {

constexpr int kMaxTop = 1024;
constexpr int kMaxCluster = 8;
constexpr int kThreads = 1536, kGradThreads = 1024;  // an SM's, at 40 and 64 registers each (the latter without the loss)
constexpr int kSlice = 64 * 1024 + 64;  // bytes of a block's slice at most, where a cluster of kMaxCluster allows it

struct Args {
    const void *teacher, *indices;
    int ttype, itype;
    int64_t ldt, ldi;
    const float *weight, *dloss, *lse_in;
    float *loss, *lse_out;
    float T;
    int64_t vocab;
    int top;
    int64_t rows;
    int slice;  // granules of a block
    uint32_t limit;  // tries of the wait for the row's other blocks
    unsigned *err;   // where one that runs out is told (null: the library's own word)
};

__device__ __forceinline__ int64_t load_index(const void *p, int it, int64_t i) {
    return it == ZPUCUDA_I64 ? ((const int64_t *)p)[i] : (int64_t)((const int32_t *)p)[i];
}

// 2^x (error 2^-22 of the result; -inf gives 0).
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// The larger of two granules' elements; a NaN among them stays.
template <typename T>
__device__ __forceinline__ uint4 max_elements(const uint4 &a, const uint4 &b) {
    uint32_t x[4] = {a.x, a.y, a.z, a.w};
    const uint32_t y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) {
            x[i] = __float_as_uint(max_nan(__uint_as_float(x[i]), __uint_as_float(y[i])));
        } else if constexpr (std::is_same<T, __half>::value) {
            const __half2 m = __hmax2_nan(*(const __half2 *)&x[i], *(const __half2 *)&y[i]);
            x[i] = *(const uint32_t *)&m;
        } else {
            const __nv_bfloat162 m = __hmax2_nan(*(const __nv_bfloat162 *)&x[i], *(const __nv_bfloat162 *)&y[i]);
            x[i] = *(const uint32_t *)&m;
        }
    }
    return make_uint4(x[0], x[1], x[2], x[3]);
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// A granule at a row's end, -inf in the place of elements outside [from, to) (counted from the granule's first).
template <typename T>
__device__ __noinline__ uint4 load_edge(const T *p, int from, int to) {
    float f[kPiece<T>];
#pragma unroll
    for (int e = 0; e < kPiece<T>; e++) f[e] = e >= from && e < to ? to_f(p[e]) : -INFINITY;
    return pack<T>(f);  // exact: the values come from that type
}

template <typename T, bool LOSS, bool GRAD, int THREADS>
__global__ void __launch_bounds__(THREADS, (LOSS ? kThreads : kGradThreads) / THREADS)
    distill_kernel(const T *logits, int64_t ld, T *out, int64_t ldo, const Args A) {
    constexpr int N = kPiece<T>, H = N / 2, WARPS = THREADS / 32, MARKS = 2048, U = 4;
    extern __shared__ __align__(16) float entries[];
    __shared__ uint64_t told;
    // each warp's largest logit, its sum of e^z relative to that, its sum of p z relative to that (to 0 where it is -inf), and
    // of p
    __shared__ float4 part[kMaxCluster * WARPS];
    __shared__ uint16_t mark[MARKS];              // an entry's number, by its place: to find indices listed twice
    __shared__ int again;
    // for each listed entry: its teacher logit / T, its logit, its place in the slice (-1: elsewhere)
    float *sp = entries, *sz = sp + A.top;
    int *si = (int *)(sz + A.top);
    uint32_t rank, size;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
    const int64_t row = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
    if (row >= A.rows) return;  // the whole cluster
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float w = A.weight ? A.weight[row] : 1.0f, dl = GRAD && A.dloss ? A.dloss[row] : 1.0f;
    const T *xr = logits + row * ld;
    // the row's granules: granule g holds elements g * N - skew + e; this block's are g0 .. g0 + n - 1, and element 0 of
    // the slice is element `base` of the row
    const int skew = (int)(((uintptr_t)xr & 15) / sizeof(T));
    const int64_t granules = (skew + A.vocab + N - 1) / N, g0 = (int64_t)rank * A.slice;
    const int n = (int)max((int64_t)0, min((int64_t)A.slice, granules - g0));
    const int64_t base = g0 * N - skew;
    const T *x = xr + base;
    T *o = GRAD ? out + row * ldo + base : nullptr;
    // the slice's elements that are in the row, its whole granules, and the partial one that this thread has
    const int from = base < 0 ? skew : 0, to = (int)max((int64_t)0, min((int64_t)n * N, A.vocab - base));
    const int w0 = from > 0, w1 = to / N;
    const int edge = threadIdx.x == 0 && w0 && n ? 0 : threadIdx.x == 32 && w1 < n && !(w0 && w1 == 0) ? w1 : -1;
    const bool same = ((uintptr_t)o & 15) == 0;  // x is on a granule: o, too?
    auto zero = [&]() {
        for (int g = w0 + threadIdx.x; g < w1; g += THREADS) {
            if (same) __stcs((uint4 *)(o + g * N), make_uint4(0, 0, 0, 0));
            else store_elements(o + g * N, make_uint4(0, 0, 0, 0), 0, N);
        }
        if (edge >= 0) store_elements(o + edge * N, make_uint4(0, 0, 0, 0), max(from - edge * N, 0), min(to - edge * N, N));
    };
    const float inv_t = 1.0f / A.T;
    if (LOSS && threadIdx.x == 0) {
        tc::mb_init(&told, size * WARPS);
        tc::mb_init_fence();
    }
    if (threadIdx.x == 0) again = 0;
    const float c = GRAD ? A.T * (w * dl) : 0.0f;
    const bool want_loss = LOSS && w != 0.0f, want_grad = GRAD && c != 0.0f, want = want_loss || want_grad;
    // the first of the row's bytes are sent for (with the loss there are no registers to spare for them), then the listed entries
    uint4 q[U];
    int g = w0 + threadIdx.x;
    auto load = [&]() {  // this thread's next U granules, -inf past its last
        constexpr uint32_t none = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
#pragma unroll
        for (int u = 0; u < U; u++)
            q[u] = g + u * THREADS < w1 ? __ldcg((const uint4 *)(x + g * N) + u * THREADS) : make_uint4(none, none, none, none);
        return g < w1;
    };
    bool more = !LOSS && want && load();
    bool bad = false;
    if (want)
        for (int k = threadIdx.x; k < A.top; k += THREADS) {
            const int64_t i = load_index(A.indices, A.itype, row * A.ldi + k);
            const float u = load_f(A.teacher, A.ttype, row * A.ldt + k) * inv_t;
            const bool in = i >= 0 && i < A.vocab;
            bad |= !in && i != -1;
            const bool here = in && i >= base && i - base < to;
            if (here) sz[k] = to_f(x[i - base]);
            si[k] = here ? (int)(i - base) : -1;
            sp[k] = in ? u : -INFINITY;
        }
    bad = __syncthreads_or(bad);  // and the barrier is ready
    float um = -INFINITY, us = 0.0f, ul = 0.0f;
    if (want)
        for (int k = lane; k < A.top; k += 32) um = max_nan(um, sp[k]);
    um = warp_max_nan(um);
    // with nothing to learn from the row (alike in all its blocks) what follows is left out
    if (want && (um != -INFINITY || bad)) {
        if (LOSS && size > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // `told` is ready
        const f32x2 k2 = make2(inv_t * 1.4426950408889634f);
        float lse = LOSS ? 0.0f : A.lse_in[row], high = 0.0f, bits = 0.0f;  // largest logit, log2 of the sum relative to it
        float4 mine;
        if constexpr (LOSS) {
            // A thread's sum is relative to its largest logit so far; a larger one scales it down first.  The distance of
            // two logits comes before 1 / T: it is exact where it counts, and does not overflow for masks of the type's
            // lowest value.
            float m = -INFINITY;
            f32x2 s2 = make2(0.0f), s3 = s2;
            auto raise = [&](const uint4 &mx) {
                float f[N], top = -INFINITY;
                unpack<T>(mx, f);
#pragma unroll
                for (int e = 0; e < N; e++) top = max_nan(top, f[e]);
                if (!(top <= m)) {
                    const float down = m == -INFINITY ? 0.0f : expf((m - top) * inv_t);
                    s2 = mul2(add2(s2, s3), make2(down));
                    s3 = make2(0.0f);
                    m = top;
                }
            };
            auto sum = [&](const uint4 &q) {
                const f32x2 neg = make2(m == -INFINITY ? 0.0f : -m);  // all -inf so far: exponentials of -inf
                f32x2 v[H];
                unpack2<T>(q, v);
#pragma unroll
                for (int e = 0; e < H; e++) {
                    const f32x2 t = mul2(add2(v[e], neg), k2), p = make2(exp2_fast(lo2(t)), exp2_fast(hi2(t)));
                    if (e & 1) s3 = add2(s3, p);
                    else s2 = add2(s2, p);
                }
            };
            more = load();
            if (edge >= 0) {
                const uint4 r = load_edge(x + edge * N, from - edge * N, to - edge * N);
                raise(r);
                sum(r);
            }
            for (; more; g += U * THREADS, more = load()) {
                uint4 mx = q[0];
#pragma unroll
                for (int u = 1; u < U; u++) mx = max_elements<T>(mx, q[u]);
                raise(mx);
#pragma unroll
                for (int u = 0; u < U; u++) sum(q[u]);
            }
            g = w0 + threadIdx.x;
            __syncwarp();
            s2 = add2(s2, s3);
            mine.x = warp_max(m);
            mine.y = warp_sum((lo2(s2) + hi2(s2)) * (m == mine.x ? 1.0f : expf((m - mine.x) * inv_t)));
        }
        for (int k = lane; k < A.top; k += 32) {
            const float d = sp[k] - um, e = expf(d);
            us += e;
            if (e != 0.0f) ul += e * d;
        }
        us = warp_sum(us);
        if (LOSS) ul = warp_sum(ul);
        const float ur = 1.0f / us;
        // the listed entries in this slice
        // (Relative to a logit of the row: z itself may be large, or a mask of the type's lowest value, and all that counts of
        // it lost in a sum with the row's log sum.)
        float pz = 0.0f, ps = 0.0f;
        const float ref = LOSS && mine.x != -INFINITY ? mine.x : 0.0f;
        for (int k = threadIdx.x; k < A.top; k += THREADS) {
            if (si[k] < 0) continue;
            const float p = expf(sp[k] - um) * ur;
            if (LOSS && p != 0.0f) {
                pz += p * ((sz[k] - ref) * inv_t);
                ps += p;
            }
            if (GRAD) mark[si[k] % MARKS] = (uint16_t)k;
        }
        bool ok = true;
        if constexpr (LOSS) {
            // Each warp tells all blocks of the row, by stores into their shared memory and one arrival, and goes on
            // when all warps of the row have: sooner than by a barrier of the whole cluster.
            mine.z = warp_sum(pz);
            mine.w = warp_sum(ps);
            if (size > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // of all blocks
            __syncwarp();
            if (lane < (int)size) {
                uint32_t there, bar;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(tc::su32(&part[rank * WARPS + warp])), "r"(lane));
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(tc::su32(&told)), "r"(lane));
                asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(there), "f"(mine.x), "f"(mine.y), "f"(mine.z),
                             "f"(mine.w)
                             : "memory");
                asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
            }
            ok = __all_sync(0xffffffffu, tc::mb_wait_cluster(&told, 0, A.err ? A.err : &g_distill_error, A.limit));
            float as = 0.0f, az = 0.0f;
            high = -INFINITY;
            for (int i = lane; i < (int)size * WARPS; i += 32) high = fmaxf(high, part[i].x);
            high = warp_max(high);
            for (int i = lane; i < (int)size * WARPS; i += 32) {
                const float4 q = part[i];
                as += q.x == high ? q.y : q.y * expf((q.x - high) * inv_t);
                if (q.w != 0.0f) az += q.z + q.w * (((q.x == -INFINITY ? 0.0f : q.x) - high) * inv_t);
            }
            as = warp_sum(as);
            bits = log2f(as);
            lse = high * inv_t + logf(as);
            if (rank == 0 && warp == 0) {
                az = warp_sum(az);
                if (lane == 0) {
                    // sum of p log p, less that of p z, plus lse, both relative to the largest logit
                    const float l = (ul * ur - logf(us)) - (az - logf(as));
                    A.loss[row] = bad || !ok ? NAN : w == 0.0f ? 0.0f : w * (A.T * A.T) * l;
                    if (A.lse_out) A.lse_out[row] = !ok ? NAN : w == 0.0f ? 0.0f : lse;
                }
            }
        } else {
            __syncthreads();  // the marks, and the entries' logits are read
        }
        if constexpr (GRAD) {
            // log2 of q: from the largest logit and the sum, or (without them) from lse, whose z is rounded like it
            auto log2q = [&](f32x2 v) {
                return LOSS ? fma2(add2(v, make2(-high)), k2, make2(-bits))
                            : mul2(add2(mul2(v, make2(inv_t)), make2(-lse)), make2(1.4426950408889634f));
            };
            const f32x2 c2 = make2(bad || !ok ? NAN : c);
            auto grad = [&](const uint4 &q) {
                f32x2 f[H];
                unpack2<T>(q, f);
#pragma unroll
                for (int e = 0; e < H; e++) {
                    const f32x2 t = log2q(f[e]);
                    f[e] = mul2(c2, make2(exp2_fast(lo2(t)), exp2_fast(hi2(t))));
                }
                return pack2<T>(f);
            };
            if (!want_grad) {
                zero();
            } else {
                if (LOSS) more = load();
                if (edge >= 0)
                    store_elements(o + edge * N, grad(load_edge(x + edge * N, from - edge * N, to - edge * N)),
                                   max(from - edge * N, 0), min(to - edge * N, N));
                for (; more; g += U * THREADS, more = load())
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        const uint4 d = grad(q[u]);
                        if (g + u * THREADS >= w1) break;
                        if (same) __stcs((uint4 *)(o + g * N) + u * THREADS, d);
                        else store_elements(o + (g + u * THREADS) * N, d, 0, N);
                    }
            }
            if (want_grad && !bad) {
                // The listed entries are written over, an index that is listed again by its first entry.
                for (int k = threadIdx.x; k < A.top; k += THREADS)
                    if (si[k] >= 0 && mark[si[k] % MARKS] != (uint16_t)k) again = 1;
                __syncthreads();
                const bool twice = again;  // perhaps: two places may share a mark
                for (int k = threadIdx.x; k < A.top; k += THREADS) {
                    const int i = si[k];
                    if (i < 0) continue;
                    float p = 0.0f;
                    bool first = true;
                    for (int j = twice ? 0 : k; j < (twice ? A.top : k + 1); j++)  // in the entries' order
                        if (si[j] == i) {
                            first &= j >= k;
                            p += expf(sp[j] - um) * ur;
                        }
                    if (first) o[i] = from_f<T>(ok ? c * (exp2_fast(lo2(log2q(make2(sz[k])))) - p) : NAN);
                }
            }
        }
        // A warp whose wait has run out stays until all have told (again with a limit), so that none of them writes to a block
        // that is gone.  (A second barrier of the cluster instead took 5 us of the loss alone, 2048 x 131072 bf16: 136 for 131.)
        if (LOSS && !ok) tc::mb_wait_cluster(&told, 0, A.err ? A.err : &g_distill_error);
        return;
    }
    if (GRAD) zero();
    if (LOSS && rank == 0 && threadIdx.x == 0) {
        A.loss[row] = 0.0f;
        if (A.lse_out) A.lse_out[row] = 0.0f;
    }
}

int check_args(const char *who, int dtype, const void *logits, int64_t ld, const Args &A, int64_t rows) {
    if (rows < 0 || A.vocab < 1) return head_error(ZPUCUDA_ERR_INVALID_SHAPE, who, "rows >= 0 and vocab >= 1 are wanted");
    if (A.vocab > 0x7fffffff || rows > 0x7fffffff)
        return head_error(ZPUCUDA_ERR_NOT_SUPPORTED, who, "more than 2^31 - 1 rows or tokens");
    if (!(A.T > 0.0f) || !isfinite(A.T))
        return head_error(ZPUCUDA_ERR_INVALID_ARGUMENT, who, "temperature is not positive and finite");
    ZC_TRY(check_matrix(who, "logits", logits, dtype, ld, rows, A.vocab));
    ZC_TRY(check_matrix(who, "teacher", A.teacher, A.ttype, A.ldt, rows, A.top));
    if (A.itype != ZPUCUDA_I32 && A.itype != ZPUCUDA_I64)
        return head_error(ZPUCUDA_ERR_NOT_SUPPORTED, who, "indices are not i32 or i64");
    ZC_TRY(check_vectors(who, A.itype == ZPUCUDA_I64 ? 8 : 4, {{"indices", A.indices}}));
    ZC_TRY(check_vectors(who, 4, {{"weight", A.weight}, {"dloss", A.dloss}, {"lse", A.lse_in}, {"loss", A.loss}, {"lse", A.lse_out}}));
    if (A.ldi < A.top) return head_error(ZPUCUDA_ERR_INVALID_SHAPE, who, "indices: row pitch below the row's length");
    if (rows > 0 && A.top > 0 && !A.indices) return head_error(ZPUCUDA_ERR_INVALID_ARGUMENT, who, "indices: null pointer");
    return ZPUCUDA_OK;
}

template <typename T, bool LOSS, bool GRAD, int THREADS>
int launch_cluster(const T *logits, int64_t ld, T *out, int64_t ldo, const Args &A, int cluster, cudaStream_t s) {
    auto f = distill_kernel<T, LOSS, GRAD, THREADS>;
    cudaLaunchConfig_t cfg = {};
    const RowGrid grid = row_grid(A.rows);
    cfg.gridDim = dim3((unsigned)cluster, grid.y, grid.z);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = 12 * (size_t)A.top;
    cfg.stream = s;
    cudaLaunchAttribute at[1] = {};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    ZC_CUDA(cudaLaunchKernelEx(&cfg, f, logits, ld, out, ldo, A));
    count_launch();
    return ZPUCUDA_OK;
}

template <typename T, bool LOSS, bool GRAD>
int launch_rows(const T *logits, int64_t ld, T *out, int64_t ldo, Args A, int64_t rows, cudaStream_t s) {
    // The blocks of a row: as few as keep slices to kSlice (what is read again has to stay in L2), or more where that
    // fills the SMs' last wave better.  A block takes about 3 us and 7 us for each 64 KiB.
    const int64_t granules = (A.vocab * (int64_t)sizeof(T) + 15) / 16 + 1, resident = (int64_t)num_sms() * ((LOSS ? kThreads : kGradThreads) / 256);
    int64_t cluster = LOSS ? (granules * 16 + kSlice - 1) / kSlice : 1;
    if (cluster > kMaxCluster) cluster = kMaxCluster;
    double best = 0.0;
    for (int64_t n = cluster; n <= kMaxCluster; n++) {
        const double t = (double)((rows * n + resident - 1) / resident) * (3.0 + 7.0 * (double)(granules * 16) / (double)(n << 16));
        if (n == cluster) best = t;
        if (n > cluster && granules * 16 < n * 8192) break;
        if (t < 0.97 * best) {
            best = t;
            cluster = n;
        }
    }
    A.rows = rows;
    A.slice = (int)((granules + cluster - 1) / cluster);
    // Short slices leave half of 256 threads without a granule: 2048 x 4000 bf16, loss and gradient, takes 21 us with 128 and
    // 28 with 256, 4096 x 500 f32 33 and 42.  Longer ones gain by them where rows are few: 37 x 32003 f32 10.6 and 10.0,
    // 64 x 8000 f32 10.0 and 8.9 (2048 x 8000 bf16 loses: 27 and 30).
    if (A.slice <= 512) return launch_cluster<T, LOSS, GRAD, 128>(logits, ld, out, ldo, A, (int)cluster, s);
    return launch_cluster<T, LOSS, GRAD, 256>(logits, ld, out, ldo, A, (int)cluster, s);
}

template <bool LOSS, bool GRAD>
int launch(const char *who, int dtype, const void *logits, int64_t ld, void *out, int64_t ldo, const Args &A,
           int64_t rows, void *stream) {
    ZC_TRY(check_args(who, dtype, logits, ld, A, rows));
    if (GRAD) ZC_TRY(check_matrix(who, "dlogits", out, dtype, ldo, rows, A.vocab));
    if (rows > 0 && LOSS && !A.loss) return head_error(ZPUCUDA_ERR_INVALID_ARGUMENT, who, "loss: null pointer");
    if (rows > 0 && GRAD && !LOSS && !A.lse_in)
        return head_error(ZPUCUDA_ERR_INVALID_ARGUMENT, who, "lse: null pointer");
    if (rows == 0) return ZPUCUDA_OK;
    if (LOSS) g_distill_waits.store(true, std::memory_order_relaxed);
    cudaStream_t s = resolve_stream(stream);
    ZC_HEAD_TYPE(dtype, T, return (launch_rows<T, LOSS, GRAD>((const T *)logits, ld, (T *)out, ldo, A, rows, s)));
}

// top is checked here, before it is narrowed.
int make_args(const char *who, Args &A, int ttype, const void *teacher, int64_t ldt, int itype, const void *indices,
              int64_t ldi, const float *weight, double temperature, int64_t vocab, int64_t top) {
    if (top < 0) return head_error(ZPUCUDA_ERR_INVALID_SHAPE, who, "top is negative");
    if (top > kMaxTop) return head_error(ZPUCUDA_ERR_NOT_SUPPORTED, who, "more than 1024 teacher entries in a row");
    A = Args{};
    A.ttype = ttype;
    A.teacher = teacher;
    A.ldt = ldt;
    A.itype = itype;
    A.indices = indices;
    A.ldi = ldi;
    A.weight = weight;
    A.T = (float)temperature;
    A.vocab = vocab;
    A.top = (int)top;
    A.limit = tc::kSpin;
    return ZPUCUDA_OK;
}

}  // namespace
}  // namespace zc

using namespace zc;

extern "C" {

int zpucuda_distill_loss(int dtype, const void *d_logits, int64_t ld, int ttype, const void *d_teacher, int64_t ldt,
                         int itype, const void *d_indices, int64_t ldi, const float *d_weight, double temperature,
                         float *d_loss, float *d_lse, int64_t rows, int64_t vocab, int64_t top, void *stream) {
    Args A;
    ZC_TRY(make_args("distill_loss", A, ttype, d_teacher, ldt, itype, d_indices, ldi, d_weight, temperature, vocab, top));
    A.loss = d_loss;
    A.lse_out = d_lse;
    return launch<true, false>("distill_loss", dtype, d_logits, ld, nullptr, 0, A, rows, stream);
}

int zpucuda_debug_distill_loss(int dtype, const void *d_logits, int64_t ld, int ttype, const void *d_teacher, int64_t ldt,
                               int itype, const void *d_indices, int64_t ldi, const float *d_weight, double temperature,
                               float *d_loss, float *d_lse, int64_t rows, int64_t vocab, int64_t top, uint32_t spin_limit,
                               uint32_t *d_err, void *stream) {
    Args A;
    ZC_TRY(make_args("debug_distill_loss", A, ttype, d_teacher, ldt, itype, d_indices, ldi, d_weight, temperature, vocab, top));
    ZC_TRY(check_vectors("debug_distill_loss", 4, {{"err", d_err}}));
    A.loss = d_loss;
    A.lse_out = d_lse;
    A.limit = spin_limit;
    A.err = d_err;
    return launch<true, false>("debug_distill_loss", dtype, d_logits, ld, nullptr, 0, A, rows, stream);
}

int zpucuda_distill_grad(int dtype, const void *d_logits, int64_t ld, int ttype, const void *d_teacher, int64_t ldt,
                         int itype, const void *d_indices, int64_t ldi, const float *d_weight, double temperature,
                         const float *d_lse, const float *d_dloss, void *d_dlogits, int64_t ldd, int64_t rows,
                         int64_t vocab, int64_t top, void *stream) {
    Args A;
    ZC_TRY(make_args("distill_grad", A, ttype, d_teacher, ldt, itype, d_indices, ldi, d_weight, temperature, vocab, top));
    A.lse_in = d_lse;
    A.dloss = d_dloss;
    return launch<false, true>("distill_grad", dtype, d_logits, ld, d_dlogits, ldd, A, rows, stream);
}

int zpucuda_distill_value_and_grad(int dtype, const void *d_logits, int64_t ld, int ttype, const void *d_teacher,
                                   int64_t ldt, int itype, const void *d_indices, int64_t ldi, const float *d_weight,
                                   double temperature, const float *d_dloss, float *d_loss, void *d_dlogits,
                                   int64_t ldd, int64_t rows, int64_t vocab, int64_t top, void *stream) {
    Args A;
    ZC_TRY(make_args("distill_value_and_grad", A, ttype, d_teacher, ldt, itype, d_indices, ldi, d_weight, temperature,
                     vocab, top));
    A.dloss = d_dloss;
    A.loss = d_loss;
    return launch<true, true>("distill_value_and_grad", dtype, d_logits, ld, d_dlogits, ldd, A, rows, stream);
}

}  // extern "C"
