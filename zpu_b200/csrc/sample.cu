// Choosing the next token of each row from given uniform numbers, with
// temperature, top-k, top-p and min-p.
//
// A token's weight is a whole number,
//   w_i = floor(2^40 * exp((x_i - max x) / T)),
// so that every sum below is exact: it does not depend on its order, and the
// same row gives the same token whatever the work's split.  Tokens are ranked
// by falling logit, equal ones by rising index.  Kept are
//   top-k:  the k first ranks;
//   top-p:  of those, the shortest run of first ranks whose weights reach
//           ceil(p * their sum);
//   min-p:  of those, the tokens with w_i >= ceil(min_p * 2^40);
// and the token is the first index whose running sum of kept weights (by
// index) exceeds floor(u * their sum).  T <= 0 takes the first rank.  A NaN
// or -inf logit has no weight; a row without any gives token -1 and log
// probability -inf.
//
// The ranks are never sorted: a set of first ranks is described by the key
// (the logit's bits in rising order) of its last member and how many of the
// tokens with that key belong to it, both found by histograms over ever
// narrower key ranges.
#include "head.cuh"

namespace zc {
namespace {

constexpr int NT = 1024, NW = NT / 32;
constexpr int NB = 2048;                 // histogram bins
constexpr uint64_t kOne = 1ull << 40;
constexpr float kSpan = 28.0f;           // w = 0 beyond (max - x) / T = 40 ln 2 = 27.73
constexpr int64_t kMaxVocab = 1 << 22;   // sums of weights stay below 2^62

struct Args {
    const void *uniform;
    int utype;
    const float *temperature;
    const int32_t *top_k;
    const float *top_p, *min_p;
    int64_t *token;
    float *logprob;
    int64_t vocab;
};

// The logit's bits as a number that rises with it; NaN is 0, below all others.
__device__ __forceinline__ uint32_t key_of(float x) {
    if (x != x) return 0;
    const uint32_t u = __float_as_uint(x + 0.0f);  // -0 and 0 are equal
    return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float((key >> 31) ? (key & 0x7fffffffu) : ~key);
}

struct Row {
    float m, inv;  // max, 1 / T
    __device__ __forceinline__ float dist(float x) const { return x == m ? 0.0f : (x - m) * inv; }
    __device__ __forceinline__ uint64_t weight(float x) const {
        if (!(x > -INFINITY)) return 0;
        if (x == m) return kOne;
        return __float2ull_rz(expf((x - m) * inv) * (float)kOne);
    }
    // Histogram bin of a logit: falling logits, rising bins; -1: no weight.
    __device__ __forceinline__ int bin(float x) const {
        const float d = -dist(x);
        return d < kSpan && x > -INFINITY ? min(NB - 1, (int)(d * ((float)NB / kSpan))) : -1;
    }
};

__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

struct Shared {
    unsigned long long mass[NB];
    unsigned long long part[NW];
    uint32_t ties[NW];
    float fmax_[NW];
    unsigned long long before, total;
    uint32_t kmin, kmax;
    int bin;
};

__device__ void clear(Shared &S) {
    __syncthreads();
    for (int i = threadIdx.x; i < NB; i += NT) S.mass[i] = 0;
    __syncthreads();
}

// The sum of the histogram.
__device__ uint64_t hist_total(Shared &S) {
    __syncthreads();
    uint64_t v = 0;
    for (int i = threadIdx.x; i < NB; i += NT) v += S.mass[i];
    v = warp_sum64(v);
    if ((threadIdx.x & 31) == 0) S.part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
    for (int i = 0; i < NW; i++) v += S.part[i];
    __syncthreads();
    return v;
}

// The first bin whose running sum reaches target (<= the total); *before: the
// sum of the bins before it.
__device__ int hist_find(Shared &S, uint64_t target, uint64_t *before) {
    __syncthreads();
    if (threadIdx.x < 32) {
        constexpr int PER = NB / 32;
        uint64_t v = 0;
        for (int i = 0; i < PER; i++) v += S.mass[threadIdx.x * PER + i];
        uint64_t inc = v;
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t t = __shfl_up_sync(0xffffffffu, inc, o);
            if (threadIdx.x >= o) inc += t;
        }
        if (inc >= target && inc - v < target) {
            uint64_t c = inc - v;
            int b = threadIdx.x * PER;
            while (c + S.mass[b] < target) c += S.mass[b++];
            S.bin = b;
            S.before = c;
        }
    }
    __syncthreads();
    *before = S.before;
    return S.bin;
}

// After a histogram over bin(): the key at which the running measure (tokens,
// or MASS: their weights) of the tokens above `floor_key` reaches target, and
// in *rem what of the measure its own tokens have to give.
template <typename T, bool MASS>
__device__ uint32_t select_key(Shared &S, const T *x, int64_t V, const Row &R, uint32_t floor_key, uint64_t target,
                               uint64_t *rem) {
    uint64_t before;
    const int b = hist_find(S, target, &before);
    target -= before;
    if (threadIdx.x == 0) {
        S.kmin = 0xffffffffu;
        S.kmax = 0;
    }
    __syncthreads();
    uint32_t lo = 0xffffffffu, hi = 0;
    for (int64_t v = threadIdx.x; v < V; v += NT) {
        const float f = to_f(x[v]);
        const uint32_t k = key_of(f);
        if (k > floor_key && R.bin(f) == b) {
            lo = min(lo, k);
            hi = max(hi, k);
        }
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if ((threadIdx.x & 31) == 0) {
        atomicMin(&S.kmin, lo);
        atomicMax(&S.kmax, hi);
    }
    __syncthreads();
    lo = S.kmin;
    hi = S.kmax;
    while (lo < hi) {
        int shift = 0;
        while (((hi - lo) >> shift) >= NB) shift++;
        clear(S);
        for (int64_t v = threadIdx.x; v < V; v += NT) {
            const float f = to_f(x[v]);
            const uint32_t k = key_of(f);
            if (k >= lo && k <= hi) atomicAdd(&S.mass[(hi - k) >> shift], MASS ? (unsigned long long)R.weight(f) : 1ull);
        }
        const int s = hist_find(S, target, &before);
        target -= before;
        hi -= (uint32_t)s << shift;
        const uint32_t width = (1u << shift) - 1;
        lo = hi - lo > width ? hi - width : lo;
    }
    *rem = target;
    return hi;
}

template <typename T>
__global__ void __launch_bounds__(NT) sample_kernel(const T *logits, int64_t ld, Args A) {
    __shared__ Shared S;
    const int64_t row = blockIdx.x, V = A.vocab;
    const T *x = logits + row * ld;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

    float m = -INFINITY;
    for (int64_t v = threadIdx.x; v < V; v += NT) m = fmaxf(m, to_f(x[v]));  // passes NaN over
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) S.fmax_[warp] = m;
    __syncthreads();
    for (int w = 0; w < NW; w++) m = fmaxf(m, S.fmax_[w]);
    if (m == -INFINITY) {
        if (threadIdx.x == 0) {
            A.token[row] = -1;
            if (A.logprob) A.logprob[row] = -INFINITY;
        }
        return;
    }
    const float temp = A.temperature ? A.temperature[row] : 1.0f;
    const Row R = {m, temp > 0.0f ? 1.0f / temp : 0.0f};

    // The kept ranks: keys above `key`, and the first `ties` tokens of that key.
    uint32_t key = 0;
    uint64_t ties = 0;
    if (!(temp > 0.0f)) {
        key = key_of(m);
        ties = 1;
    } else {
        const int64_t k = A.top_k ? A.top_k[row] : 0;
        if (k > 0 && k < V) {
            clear(S);
            for (int64_t v = threadIdx.x; v < V; v += NT) {
                const int b = R.bin(to_f(x[v]));
                if (b >= 0) atomicAdd(&S.mass[b], 1ull);
            }
            if (hist_total(S) > (uint64_t)k) key = select_key<T, false>(S, x, V, R, 0, (uint64_t)k, &ties);
        }
        const float p = A.top_p ? A.top_p[row] : 1.0f;
        if (p < 1.0f) {
            clear(S);
            for (int64_t v = threadIdx.x; v < V; v += NT) {
                const float f = to_f(x[v]);
                const int b = R.bin(f);
                if (b >= 0 && key_of(f) > key) atomicAdd(&S.mass[b], (unsigned long long)R.weight(f));
            }
            const uint64_t above = hist_total(S), wk = key ? R.weight(value_of(key)) : 0;
            const double edge = ceil((double)p * (double)(int64_t)(above + ties * wk));
            const uint64_t target = edge >= 1.0 ? (uint64_t)edge : 1;
            if (above >= target) {
                uint64_t rem;
                key = select_key<T, true>(S, x, V, R, key, target, &rem);
                const uint64_t w = R.weight(value_of(key));
                ties = (rem + w - 1) / w;
            } else {
                const uint64_t need = (target - above + wk - 1) / wk;  // wk > 0: the total is above `above`
                ties = need < ties ? need : ties;
            }
        }
    }
    uint64_t least = 0;
    const float mp = A.min_p ? A.min_p[row] : 0.0f;
    if (mp > 0.0f) least = mp < 1.0f ? (uint64_t)ceil((double)mp * (double)kOne) : kOne;

    // Running sums by index: a segment for each warp.
    uint64_t wk = key ? R.weight(value_of(key)) : 0;
    if (wk < least) wk = 0;
    const int64_t seg = (V + NT - 1) / NT * 32, v0 = warp * seg, v1 = v0 + seg < V ? v0 + seg : V;
    auto kept = [&](float f) -> uint64_t {
        if (key_of(f) <= key) return 0;
        const uint64_t w = R.weight(f);
        return w >= least ? w : 0;
    };
    uint64_t sum = 0;
    uint32_t same = 0;
    for (int64_t v = v0 + lane; v < v1; v += 32) {
        const float f = to_f(x[v]);
        sum += kept(f);
        same += key && key_of(f) == key;
    }
    sum = warp_sum64(sum);
    same = __reduce_add_sync(0xffffffffu, same);
    __syncthreads();
    if (lane == 0) {
        S.part[warp] = sum;
        S.ties[warp] = same;
    }
    __syncthreads();
    uint64_t total = 0, left = ties;
    for (int w = 0; w < NW; w++) {
        const uint64_t t = S.ties[w] < left ? S.ties[w] : left;
        left -= t;
        total += S.part[w] + t * wk;
    }
    const double u = A.utype == ZPUCUDA_F64 ? ((const double *)A.uniform)[row] : (double)((const float *)A.uniform)[row];
    uint64_t at = 0;
    if (u > 0.0) {
        const double r = floor(u * (double)(int64_t)total);
        at = r < (double)(int64_t)total ? (uint64_t)r : total;
        if (at >= total) at = total - 1;
    }
    uint64_t before = 0;
    left = ties;
    for (int w = 0; w < warp; w++) {
        const uint64_t t = S.ties[w] < left ? S.ties[w] : left;
        left -= t;
        before += S.part[w] + t * wk;
    }
    const uint64_t mine = S.part[warp] + (S.ties[warp] < left ? S.ties[warp] : left) * wk;
    if (at < before || at >= before + mine) return;
    for (int64_t v = v0; v < v1; v += 32) {
        const float f = v + lane < v1 ? to_f(x[v + lane]) : -INFINITY;
        const bool eq = key && key_of(f) == key;
        const uint32_t eqs = __ballot_sync(0xffffffffu, eq);
        uint64_t w = kept(f);
        if (eq && __popc(eqs & ((1u << lane) - 1)) < left) w = wk;
        uint64_t inc = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += t;
        }
        const uint32_t over = __ballot_sync(0xffffffffu, before + inc > at);
        if (over) {
            if (lane == __ffs(over) - 1) {
                A.token[row] = v + lane;
                if (A.logprob) A.logprob[row] = R.dist(f) - logf((float)(int64_t)total / (float)kOne);
            }
            return;
        }
        before += __shfl_sync(0xffffffffu, inc, 31);
        const uint64_t n = __popc(eqs);
        left -= n < left ? n : left;
    }
}

}  // namespace
}  // namespace zc

using namespace zc;

extern "C" int zpucuda_sample(int dtype, const void *d_logits, int64_t ld, int utype, const void *d_uniform,
                              const float *d_temperature, const int32_t *d_top_k, const float *d_top_p,
                              const float *d_min_p, int64_t *d_token, float *d_logprob, int64_t rows, int64_t vocab,
                              void *stream) {
    if (rows < 0 || vocab < 1) return set_error(ZPUCUDA_ERR_INVALID_SHAPE, "sample: rows >= 0 and vocab >= 1 are wanted");
    if (vocab > kMaxVocab) return set_error(ZPUCUDA_ERR_NOT_SUPPORTED, "sample: more than 2^22 tokens");
    if (rows > 0x7fffffff) return set_error(ZPUCUDA_ERR_NOT_SUPPORTED, "sample: more than 2^31 - 1 rows");
    ZC_TRY(check_matrix("sample", "logits", d_logits, dtype, ld, rows, vocab));
    if (utype != ZPUCUDA_F32 && utype != ZPUCUDA_F64) return set_error(ZPUCUDA_ERR_NOT_SUPPORTED, "sample: uniform is not f32 or f64");
    if (rows == 0) return ZPUCUDA_OK;
    if (!d_uniform || !d_token) return set_error(ZPUCUDA_ERR_INVALID_ARGUMENT, "sample: uniform or token: null pointer");
    const Args A = {d_uniform, utype, d_temperature, d_top_k, d_top_p, d_min_p, d_token, d_logprob, vocab};
    cudaStream_t s = resolve_stream(stream);
    ZC_HEAD_TYPE(dtype, T, sample_kernel<T><<<(unsigned)rows, NT, 0, s>>>((const T *)d_logits, ld, A));
    ZC_LAUNCHED("sample_kernel");
    return ZPUCUDA_OK;
}
