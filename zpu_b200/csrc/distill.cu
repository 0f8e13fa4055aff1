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
#include "head.cuh"

namespace zc {
namespace {

constexpr int NT = 256;
constexpr int kMaxTop = 1024;

struct Args {
    const void *teacher, *indices;
    int ttype, itype;
    int64_t ldt, ldi;
    const float *weight, *dloss, *lse_in;
    float *loss, *lse_out;
    float T;
    int64_t vocab;
    int top;
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

template <typename T, bool LOSS, bool GRAD>
__global__ void __launch_bounds__(NT) distill_kernel(const T *logits, int64_t ld, T *out, int64_t ldo, Args A) {
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
    ZC_HEAD_TYPE(dtype, T,
                 (distill_kernel<T, LOSS, GRAD>
                  <<<(unsigned)rows, NT, 0, s>>>((const T *)logits, ld, (T *)out, ldo, A)));
    ZC_LAUNCHED("distill_kernel");
    return ZPUCUDA_OK;
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
