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
// element where both loss and gradient are wanted): a row is copied once into
// the shared memory of a cluster of blocks, a slice each, where its maximum, sum
// and gradient are computed; slices are small enough (64 KiB) that several
// blocks of an SM overlap one another's copies and arithmetic.  A slice is
// counted in aligned 16-byte granules of memory, so an odd vocabulary costs two
// partial granules a row and nothing else.
#include "head.cuh"
#include "tcgen05.cuh"
#include "waits.cuh"

namespace zc {

static __device__ unsigned int g_distill_error;

int distill_device_error(unsigned int *e) {
    ZC_CUDA(cudaMemcpyFromSymbol(e, g_distill_error, sizeof *e));
    return ZPUCUDA_OK;
}

namespace {

constexpr int NT = 256;
constexpr int kMaxTop = 1024;
constexpr int kMaxCluster = 8;
constexpr int kSlice = 66 * 1024, kMaxSlice = 200 * 1024;  // bytes: wanted (three blocks an SM), possible
constexpr int kCopies = 4;                                 // of a slice, each waited for by itself

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
    int slice_bytes;  // of a block's shared memory
};

__device__ __forceinline__ int64_t load_index(const void *p, int it, int64_t i) {
    return it == ZPUCUDA_I64 ? ((const int64_t *)p)[i] : (int64_t)((const int32_t *)p)[i];
}

__device__ __forceinline__ float block_max(float v, float *sm) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sm[0];
#pragma unroll
    for (int w = 1; w < NT / 32; w++) v = fmaxf(v, sm[w]);
    return v;
}
__device__ __forceinline__ float block_sum(float v, float *sm) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < NT / 32; w++) v += sm[w];
    return v;
}

// 2^x (error 2^-22 of the result; -inf gives 0).
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// The larger of two granules' elements, NaN passed over.
template <typename T>
__device__ __forceinline__ uint4 max_elements(const uint4 &a, const uint4 &b) {
    uint32_t x[4] = {a.x, a.y, a.z, a.w};
    const uint32_t y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) {
            x[i] = __float_as_uint(fmaxf(__uint_as_float(x[i]), __uint_as_float(y[i])));
        } else if constexpr (std::is_same<T, __half>::value) {
            const __half2 m = __hmax2(*(const __half2 *)&x[i], *(const __half2 *)&y[i]);
            x[i] = *(const uint32_t *)&m;
        } else {
            const __nv_bfloat162 m = __hmax2(*(const __nv_bfloat162 *)&x[i], *(const __nv_bfloat162 *)&y[i]);
            x[i] = *(const uint32_t *)&m;
        }
    }
    return make_uint4(x[0], x[1], x[2], x[3]);
}

// exp2 arguments of a granule relative to `ref`.  16-bit logits take one
// multiply-add (k = log2(e) / T, its rounding is far below theirs); 32-bit ones
// form z - ref first, so that the error stays relative to the distance.
template <typename T>
struct Scale {
    f32x2 k, off, log2e;
    __device__ __forceinline__ Scale(float inv_t, float ref) {
        if constexpr (sizeof(T) == 4) {
            k = make2(inv_t);
            off = make2(-ref);
            log2e = make2(1.4426950408889634f);
        } else {
            k = make2(inv_t * 1.4426950408889634f);
            off = make2(-ref * 1.4426950408889634f);
        }
    }
    __device__ __forceinline__ f32x2 arg(f32x2 x) const {
        const f32x2 d = fma2(x, k, off);
        if constexpr (sizeof(T) == 4) return mul2(d, log2e);
        else return d;
    }
};

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// The first waits of a block must not be the last: several blocks share an SM,
// and what one waits for another's arithmetic hides, but each byte of shared
// memory is held from its copy to its gradient, so HBM's bandwidth needs a short
// way from one to the other.  Hence: the listed entries are fetched while the
// copies are on their way, every warp works out the teacher's sums for itself, and
// the warps of a row's blocks exchange their maxima and sums directly, by stores
// to one another's shared memory and one arrival, without a barrier of all.
template <typename T, bool LOSS, bool GRAD, int THREADS>
__global__ void __launch_bounds__(THREADS, 768 / THREADS)
    distill_kernel(const T *logits, int64_t ld, T *out, int64_t ldo, const Args A) {
    constexpr int N = kPiece<T>, WARPS = THREADS / 32, MARKS = 2048;
    extern __shared__ __align__(128) uint4 slice_smem[];
    __shared__ uint64_t full[kCopies], told;
    __shared__ float4 part[kMaxCluster * WARPS];  // each warp's maximum of z, sum of e^(z - maximum), sum of p z
    __shared__ uint16_t mark[MARKS];              // an entry's number, by its place: to find indices listed twice
    __shared__ int again;
    // behind the slice, for each listed entry: its probability, its logit, its place in the slice (-1: elsewhere)
    float *sp = (float *)((uint8_t *)slice_smem + A.slice_bytes), *sz = sp + A.top;
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
    const int64_t granules = (skew + A.vocab + N - 1) / N, g0 = (int64_t)rank * (A.slice_bytes / 16);
    const int n = (int)max((int64_t)0, min((int64_t)(A.slice_bytes / 16), granules - g0));
    const int64_t base = g0 * N - skew;
    const T *x = xr + base;
    T *o = GRAD ? out + row * ldo + base : nullptr;
    // the slice's elements that are in the row, and its granules that are whole
    const int from = base < 0 ? skew : 0, to = (int)max((int64_t)0, min((int64_t)n * N, A.vocab - base));
    const int w0 = from > 0, w1 = to / N;
    const float inv_t = 1.0f / A.T;
    const int per = (n + kCopies - 1) / kCopies;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kCopies; i++) tc::mb_init(&full[i], 1);
        tc::mb_init(&told, size * WARPS);
        tc::mb_init_fence();
        again = 0;
    }
    const float c = GRAD ? A.T * (w * dl) : 0.0f;
    const bool want_loss = LOSS && w != 0.0f, want_grad = GRAD && c != 0.0f, want = want_loss || want_grad;

    // the whole granules by bulk copies, the others element by element
    if (want) {
        if (threadIdx.x == 0)
            for (int i = 0; i < kCopies; i++) {
                const int a = max(i * per, w0), b = min(i * per + per, w1);
                const uint32_t bytes = a < b ? (uint32_t)(b - a) * 16 : 0;
                tc::mb_expect_tx(&full[i], bytes);
                if (bytes)
                    asm volatile(
                        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                            tc::su32(slice_smem + a)),
                        "l"(x + (int64_t)a * N), "r"(bytes), "r"(tc::su32(&full[i]))
                        : "memory");
            }
        if (threadIdx.x < N && w0) {
            const int e = threadIdx.x;
            ((T *)slice_smem)[e] = e >= from && e < to ? x[e] : from_f<T>(-INFINITY);
        }
        if (threadIdx.x >= 32 && threadIdx.x < 32 + N && w1 < n && !(w0 && w1 == 0)) {
            const int e = w1 * N + threadIdx.x - 32;
            ((T *)slice_smem)[e] = e < to ? x[e] : from_f<T>(-INFINITY);
        }
    }
    // the listed entries
    bool bad = false;
    if (want)
        for (int k = threadIdx.x; k < A.top; k += THREADS) {
            const int64_t i = load_index(A.indices, A.itype, row * A.ldi + k);
            const float u = load_f(A.teacher, A.ttype, row * A.ldt + k) * inv_t;
            const bool in = i >= 0 && i < A.vocab;
            bad |= !in && i != -1;
            si[k] = in && i >= base && i - base < to ? (int)(i - base) : -1;
            sp[k] = in ? u : -INFINITY;
        }
    bad = __syncthreads_or(bad);  // the entries, the barriers and the partial granules are in place
    float um = -INFINITY, us = 0.0f, ul = 0.0f;
    if (want)
        for (int k = lane; k < A.top; k += 32) um = max_nan(um, sp[k]);
    um = warp_max_nan(um);
    // with nothing to learn from the row (alike in all its blocks) what follows is left out
    if (want && (um != -INFINITY || bad)) {
        if (LOSS && size > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // `told` is ready
        for (int k = lane; k < A.top; k += 32) {
            const float d = sp[k] - um, e = expf(d);
            us += e;
            if (e != 0.0f) ul += e * d;
        }
        us = warp_sum(us);
        if (LOSS) ul = warp_sum(ul);
        const float ur = 1.0f / us;
        bool ok = true, any = false;
        uint4 mx = make_uint4(0, 0, 0, 0);
        int landed = 0, copy = 0;
        if (LOSS)
            for (int g = threadIdx.x; g < n; g += THREADS) {
                for (; g >= landed; landed += per, copy++)
                    if (!tc::mb_wait(&full[copy], 0, &g_distill_error)) ok = false;
                const uint4 q = slice_smem[g];
                mx = any ? max_elements<T>(mx, q) : q;
                any = true;
            }
        for (; copy < kCopies; copy++)
            if (!tc::mb_wait(&full[copy], 0, &g_distill_error)) ok = false;
        __syncwarp();
        float lse = LOSS ? 0.0f : A.lse_in[row];
        float4 mine;
        if constexpr (LOSS) {
            float f[N], m = -INFINITY;
            unpack<T>(mx, f);
            if (any)
#pragma unroll
                for (int e = 0; e < N; e++) m = fmaxf(m, f[e]);
            mine.x = fmaxf(warp_max(m) * inv_t, -3.0e38f);  // a slice of -inf has a sum of 0
            const Scale<T> sc(inv_t, mine.x);
            f32x2 s2 = make2(0.0f), s3 = s2;
#pragma unroll 4
            for (int g = threadIdx.x; g < n; g += THREADS) {
                f32x2 v[N / 2];
                unpack2<T>(slice_smem[g], v);
#pragma unroll
                for (int e = 0; e < N / 2; e++) {
                    const f32x2 t = sc.arg(v[e]), q = make2(exp2_fast(lo2(t)), exp2_fast(hi2(t)));
                    if (e & 1) s3 = add2(s3, q);
                    else s2 = add2(s2, q);
                }
            }
            __syncwarp();
            s2 = add2(s2, s3);
            mine.y = warp_sum(lo2(s2) + hi2(s2));
        }
        // the listed entries in this slice
        float pz = 0.0f;
        for (int k = threadIdx.x; k < A.top; k += THREADS) {
            if (si[k] < 0) continue;
            const float p = expf(sp[k] - um) * ur, z = to_f(((const T *)slice_smem)[si[k]]);
            sz[k] = z;
            if (LOSS && p != 0.0f) pz += p * (z * inv_t);
            if (GRAD) mark[si[k] % MARKS] = (uint16_t)k;
        }
        if constexpr (LOSS) {
            mine.z = warp_sum(pz);
            mine.w = 0.0f;
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
            if (!tc::mb_wait_cluster(&told, 0, &g_distill_error)) ok = false;
            __syncwarp();
            float am = -INFINITY, as = 0.0f, az = 0.0f;
            for (int i = lane; i < (int)size * WARPS; i += 32) am = fmaxf(am, part[i].x);
            am = warp_max(am);
            for (int i = lane; i < (int)size * WARPS; i += 32) {
                const float4 q = part[i];
                as += q.y * expf(q.x - am);
                az += q.z;
            }
            lse = am + logf(warp_sum(as));
            if (rank == 0 && warp == 0) {
                az = warp_sum(az);
                if (lane == 0) {
                    // sum of p log p, less that of p z, plus lse
                    const float l = (ul * ur - logf(us)) - (az - lse);
                    A.loss[row] = bad || !ok ? NAN : w == 0.0f ? 0.0f : w * (A.T * A.T) * l;
                    if (A.lse_out) A.lse_out[row] = w == 0.0f ? 0.0f : lse;
                }
            }
        } else {
            __syncthreads();  // the marks
        }
        if constexpr (GRAD) {
            const Scale<T> sc(inv_t, lse);
            const f32x2 c2 = make2(bad || !ok ? NAN : c);
            const bool same = ((uintptr_t)o & 15) == 0;  // x is on a granule: o, too?
            if (want_grad && same) {
#pragma unroll 2
                for (int g = threadIdx.x; g < n; g += THREADS) {
                    f32x2 f[N / 2];
                    unpack2<T>(slice_smem[g], f);
#pragma unroll
                    for (int e = 0; e < N / 2; e++) {
                        const f32x2 t = sc.arg(f[e]);
                        f[e] = mul2(c2, make2(exp2_fast(lo2(t)), exp2_fast(hi2(t))));
                    }
                    const uint4 q = pack2<T>(f);
                    if (g >= w0 && g < w1) *(uint4 *)(o + g * N) = q;
                    else store_elements(o + g * N, q, max(from - g * N, 0), min(to - g * N, N));
                }
            } else {
                for (int g = threadIdx.x; g < n; g += THREADS) {
                    f32x2 f[N / 2];
                    unpack2<T>(slice_smem[g], f);
#pragma unroll
                    for (int e = 0; e < N / 2; e++) {
                        const f32x2 t = sc.arg(f[e]);
                        f[e] = want_grad ? mul2(c2, make2(exp2_fast(lo2(t)), exp2_fast(hi2(t)))) : make2(0.0f);
                    }
                    store_elements(o + g * N, pack2<T>(f), max(from - g * N, 0), min(to - g * N, N));
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
                    if (first) o[i] = from_f<T>(ok ? c * (exp2_fast(lo2(sc.arg(make2(sz[k])))) - p) : NAN);
                }
            }
        }
        if (!ok)  // give up only once the copies in flight have landed
            for (int i = 0; i < kCopies; i++) tc::mb_wait(&full[i], 0, &g_distill_error);
        return;
    }
    if (want)  // the copies are on their way: not before they have landed
        for (int i = 0; i < kCopies; i++) tc::mb_wait(&full[i], 0, &g_distill_error);
    if (GRAD)
        for (int g = threadIdx.x; g < n; g += THREADS) {
            if (((uintptr_t)o & 15) == 0 && g >= w0 && g < w1) *(uint4 *)(o + g * N) = make_uint4(0, 0, 0, 0);
            else store_elements(o + g * N, make_uint4(0, 0, 0, 0), max(from - g * N, 0), min(to - g * N, N));
        }
    if (LOSS && rank == 0 && threadIdx.x == 0) {
        A.loss[row] = 0.0f;
        if (A.lse_out) A.lse_out[row] = 0.0f;
    }
}

// Rows that no cluster holds, read three times.
template <typename T, bool LOSS, bool GRAD>
__global__ void __launch_bounds__(NT) distill_long_kernel(const T *logits, int64_t ld, T *out, int64_t ldo, Args A) {
    __shared__ float sm[NT / 32];
    __shared__ float sp[kMaxTop], sz[kMaxTop];
    __shared__ int si[kMaxTop];
    const int64_t row = blockIdx.x;
    const T *x = logits + row * ld;
    T *o = GRAD ? out + row * ldo : nullptr;
    const float w = A.weight ? A.weight[row] : 1.0f;
    const float c = GRAD ? A.T * (w * (A.dloss ? A.dloss[row] : 1.0f)) : 0.0f;
    const bool want_loss = LOSS && w != 0.0f, want_grad = GRAD && c != 0.0f;

    // the teacher's distribution
    float um = -INFINITY;
    bool bad = false;
    if (want_loss || want_grad)
        for (int k = threadIdx.x; k < A.top; k += NT) {
            const int64_t i = load_index(A.indices, A.itype, row * A.ldi + k);
            const bool in = i >= 0 && i < A.vocab;
            bad |= !in && i != -1;
            const float u = in ? load_f(A.teacher, A.ttype, row * A.ldt + k) / A.T : -INFINITY;
            si[k] = in ? (int)i : -1;
            sp[k] = u;
            sz[k] = in ? to_f(x[i]) / A.T : 0.0f;
            um = max_nan(um, u);
        }
    bad = __syncthreads_or(bad);
    const bool un = __syncthreads_or(um != um);
    um = un ? NAN : block_max(um, sm);
    if (!(want_loss || want_grad) || (um == -INFINITY && !bad)) {
        if (GRAD)
            for (int64_t v = threadIdx.x; v < A.vocab; v += NT) o[v] = from_f<T>(0.0f);
        if (LOSS && threadIdx.x == 0) {
            A.loss[row] = 0.0f;
            if (A.lse_out) A.lse_out[row] = 0.0f;
        }
        return;
    }
    float us = 0.0f;
    for (int k = threadIdx.x; k < A.top; k += NT) us += expf(sp[k] - um);
    us = block_sum(us, sm);
    const float lus = logf(us);

    // the student's normaliser
    float lse;
    if (LOSS) {
        float m = -INFINITY, s = 0.0f;
        for (int64_t v = threadIdx.x; v < A.vocab; v += NT) m = fmaxf(m, to_f(x[v]) / A.T);
        m = block_max(m, sm);
        for (int64_t v = threadIdx.x; v < A.vocab; v += NT) s += expf(to_f(x[v]) / A.T - m);
        lse = m + logf(block_sum(s, sm));
    } else {
        lse = A.lse_in[row];
    }
    if (LOSS) {
        float l = 0.0f;
        for (int k = threadIdx.x; k < A.top; k += NT) {
            const float lp = (sp[k] - um) - lus, p = expf(sp[k] - um) / us;
            if (p != 0.0f) l += p * (lp - (sz[k] - lse));
        }
        l = block_sum(l, sm);
        if (threadIdx.x == 0) {
            A.loss[row] = bad ? NAN : w == 0.0f ? 0.0f : w * (A.T * A.T) * l;
            if (A.lse_out) A.lse_out[row] = lse;
        }
    }
    if (!GRAD) return;
    for (int64_t v = threadIdx.x; v < A.vocab; v += NT)
        o[v] = from_f<T>(bad ? NAN : c == 0.0f ? 0.0f : c * expf(to_f(x[v]) / A.T - lse));
    if (bad || c == 0.0f) return;
    for (int k = threadIdx.x; k < A.top; k += NT) sp[k] = expf(sp[k] - um) / us;
    __syncthreads();
    // the listed entries; an index that is listed again is written by its first entry
    for (int k = threadIdx.x; k < A.top; k += NT) {
        const int i = si[k];
        if (i < 0) continue;
        float p = 0.0f;
        bool first = true;
        for (int j = 0; j < A.top; j++)
            if (si[j] == i) {
                if (j < k) first = false;
                p += sp[j];
            }
        if (first) o[i] = from_f<T>(c * (expf(sz[k] - lse) - p));
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
    if (A.ldi < A.top) return head_error(ZPUCUDA_ERR_INVALID_SHAPE, who, "indices: row pitch below the row's length");
    if (rows > 0 && A.top > 0 && !A.indices) return head_error(ZPUCUDA_ERR_INVALID_ARGUMENT, who, "indices: null pointer");
    return ZPUCUDA_OK;
}

template <typename T, bool LOSS, bool GRAD, int THREADS>
int launch_cluster(const T *logits, int64_t ld, T *out, int64_t ldo, const Args &A, int cluster, cudaStream_t s) {
    auto f = distill_kernel<T, LOSS, GRAD, THREADS>;
    static bool attr[64] = {false};
    const int dev = current_device();
    if (dev < 0 || dev >= 64 || !attr[dev]) {
        ZC_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSlice + 16 + 12 * kMaxTop));
        if (dev >= 0 && dev < 64) attr[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    const int64_t y = A.rows < 32768 ? A.rows : 32768;
    cfg.gridDim = dim3((unsigned)cluster, (unsigned)y, (unsigned)((A.rows + y - 1) / y));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = (size_t)A.slice_bytes + 12 * (size_t)A.top;
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
    // slices of kSlice bytes at most while a cluster allows it; smaller ones while blocks are few
    const int64_t granules = (A.vocab * (int64_t)sizeof(T) + 15) / 16 + 1;
    int64_t cluster = (granules * 16 + kSlice - 1) / kSlice;
    while (cluster < kMaxCluster && rows * cluster < 2 * (int64_t)num_sms() && granules * 16 > cluster * 16384) cluster++;
    if (cluster > kMaxCluster) cluster = kMaxCluster;
    const int64_t slice = (granules + cluster - 1) / cluster * 16;
    if (slice > kMaxSlice) {
        distill_long_kernel<T, LOSS, GRAD><<<(unsigned)rows, NT, 0, s>>>(logits, ld, out, ldo, A);
        ZC_LAUNCHED("distill_long_kernel");
        return ZPUCUDA_OK;
    }
    A.rows = rows;
    A.slice_bytes = (int)slice;
    if (slice <= 8192) return launch_cluster<T, LOSS, GRAD, 128>(logits, ld, out, ldo, A, (int)cluster, s);
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
