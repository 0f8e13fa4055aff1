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
// A set of first ranks is described by the key (the logit's bits in rising order)
// of its last member and how many of the tokens with that key belong to it.  The
// vocabulary is never sorted.  One block takes a row, which stays in L2 between
// its passes, read 16 bytes at a time:
//   - Few first ranks (top_k up to kQuick): the k-th largest of the threads' own
//     maxima is a bound that at least k tokens reach and few more do; those are
//     listed and sorted, and the rest of the row is not looked at again.
//   - Otherwise a histogram of exact weights (or counts) over the logits' distance
//     from the largest finds the bin in which the set ends, and that bin's tokens are
//     listed and sorted.  What weighs too little to reach into the set is left out.
//   - 16-bit logits have few values: a count of each takes the place of the weights'
//     histogram, so only the values' weights are computed, not the tokens'.
// Two blocks of 512 threads share an SM where there are enough rows, otherwise a row
// has 1024 threads (64 x 32000 f16, top_p: 36 us, with 512 42 us).
//
// Instructions bound it, not HBM: one to find the largest; to count a value a dozen
// and an addition in shared memory, whose banks bound that pass; two dozen with an
// exponential to sum the kept weights.  256 x 131071 bf16 (67 MB) takes 16 us
// without temperature, 30 with top_k 50, 51 without a rule, 88 with top_p 0.9; 256 x
// 50000 f32 with top_p 0.9 takes 71 (weights in four parts of 10 bits, an addition
// in shared memory each).
#include <cstring>

#include "head.cuh"

namespace zc {
namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;  // of a block at most
constexpr int NB = 2048;                 // histogram bins
constexpr int kList = 4096;              // tokens listed at most
// First ranks that the threads' maxima bound well.  With 512 threads a row, 256 x 131071 bf16 takes 30 us at 50, 57 at 300 and
// 86 at 400, by histogram 84; with 1024, 1 x 131071 takes 34 us at 400, by histogram 43.
constexpr int kQuick = 400;
constexpr uint64_t kOne = 1ull << 40;
constexpr int kPlaces = 20 * 1024;       // values of 16-bit logits in the table
constexpr int kNear = 2048;              // logits about zero listed at most
constexpr float kSpan = 28.0f;           // w = 0 beyond (max - x) / T = 40 ln 2 = 27.73
constexpr int64_t kMaxVocab = (1 << 22) - 1;  // sums of weights stay below 2^62, of their 10-bit digits below 2^32

struct Args {
    const void *uniform;
    int utype;
    const float *temperature;
    const int32_t *top_k;
    const float *top_p, *min_p;
    int64_t *token;
    float *logprob;
    int64_t vocab;
    int places;  // of the table of values
};

__device__ __forceinline__ int NT() { return (int)blockDim.x; }
__device__ __forceinline__ int NW() { return (int)blockDim.x >> 5; }

// The logit's bits as a number that rises with it; NaN is 0, below all others.
__device__ __forceinline__ uint32_t key_of(float x) {
    if (x != x) return 0;
    const uint32_t u = __float_as_uint(x + 0.0f);  // -0 and 0 are equal
    return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float((key >> 31) ? (key & 0x7fffffffu) : ~key);
}

__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// The sum of the values of this lane and those below it.
__device__ __forceinline__ uint64_t warp_scan64(uint64_t v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    return v;
}

// Dynamic shared memory: one of the three at a time.
extern __shared__ __align__(16) uint32_t sample_smem[];
constexpr size_t kSmem = 4 * NB * sizeof(uint32_t);
static_assert(kSmem >= kList * sizeof(unsigned long long) && kPlaces * sizeof(uint32_t) >= kSmem, "shared memory");
// a histogram: 10 bits of the weights each (a count: the first)
__device__ __forceinline__ uint32_t &digit(int i, int b) { return sample_smem[i * NB + b]; }
// tokens as key << 32 | ~index: sorted falling, ranks
__device__ __forceinline__ unsigned long long &list(int i) { return ((unsigned long long *)sample_smem)[i]; }

struct Shared {
    unsigned long long w[kThreads];
    unsigned long long part[kWarps];
    uint32_t ties[kWarps];
    float fmax_[kWarps];
    unsigned long long before;
    uint32_t kmin, kmax;
    int bin, count;
    uint4 edge[2];  // the row's first and last granule, if they reach past it
};

// A row in granules of 16 aligned bytes, warp w's from w * seg on; and its weights.
template <typename T>
struct Row {
    static constexpr int N = kPiece<T>;
    const T *x;   // granule 0 (which may begin before the row)
    int skew, n;  // elements of granule 0 before the row, granules
    int64_t vocab;
    int seg, g0, g1, lane;  // granules of a warp, this warp's
    int first, last;        // the granules that lie in the row as a whole
    const uint4 *edge;      // the others, -inf outside the row
    float m, inv;           // the largest logit, 1 / T (0: the largest alone)

    __device__ __forceinline__ uint4 load_edge(int g) const {
        const int64_t at = (int64_t)g * N - skew;
        float f[N];
#pragma unroll
        for (int e = 0; e < N; e++) f[e] = at + e >= 0 && at + e < vocab ? to_f(x[(int64_t)g * N + e]) : -INFINITY;
        return pack<T>(f);  // exact: the values come from that type
    }
    __device__ __forceinline__ uint4 load(int g) const {
        return g >= first && g < last ? __ldcg((const uint4 *)(x + (int64_t)g * N)) : edge[g >= first];
    }
    // f(granule's bytes, its number) for each of this lane's granules from a to b, U loads in flight; lanes past the end
    // are left out.
    template <int U = 2, typename F>
    __device__ __forceinline__ void each(int a, int b, F f) const {
        for (int g = a + lane; g < b; g += 32 * U) {
            uint4 q[U];
#pragma unroll
            for (int u = 0; u < U; u++)
                if (g + 32 * u < b) q[u] = load(g + 32 * u);
#pragma unroll
            for (int u = 0; u < U; u++)
                if (g + 32 * u < b) f(q[u], g + 32 * u);
        }
        __syncwarp();
    }
    static __device__ __forceinline__ float largest(const uint4 &q) {  // passes NaN over
        if constexpr (sizeof(T) == 2) {
            using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
            T2 h[4];
            memcpy(h, &q, 16);
            const T2 t = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
            return fmaxf(fmaxf(-INFINITY, to_f(t.x)), to_f(t.y));
        }
        float f[N], t = -INFINITY;
        unpack<T>(q, f);
#pragma unroll
        for (int e = 0; e < N; e++) t = fmaxf(t, f[e]);
        return t;
    }
    __device__ __forceinline__ float dist(float f) const { return f == m ? 0.0f : (f - m) * inv; }
    bool spike;  // only the largest logit has weight: it is infinite, or 1 / T is
    __device__ __forceinline__ uint64_t weight(float f) const {
        if (spike) return f == m ? kOne : 0;
        const float d = (f - m) * inv;
        return d > -kSpan + 0.2f ? weigh_bits(__float_as_uint(expf(d))) : 0;  // NaN: 0
    }
    __device__ __forceinline__ int64_t index(int g, int e) const { return (int64_t)g * N + e - skew; }
};

__device__ __forceinline__ unsigned long long entry_of(uint32_t key, int64_t index) {
    return (unsigned long long)key << 32 | (uint32_t)~(uint32_t)index;
}
__device__ __forceinline__ uint32_t entry_key(unsigned long long e) { return (uint32_t)(e >> 32); }
__device__ __forceinline__ uint32_t entry_index(unsigned long long e) { return ~(uint32_t)e; }

// The list's n entries in falling order.
__device__ void sort_list(int n) {
    if (n <= 2 * NT()) {  // each to the place of its rank
        __syncthreads();
        const int i = threadIdx.x, j = i + NT();
        const unsigned long long a = i < n ? list(i) : 0, b = j < n ? list(j) : 0;
        int ra = 0, rb = 0;
        if (n <= NT()) {
            if (i < n)
#pragma unroll 4
                for (int k = 0; k < n; k++) ra += list(k) > a;
        } else {
#pragma unroll 4
            for (int k = 0; k < n; k++) {
                const unsigned long long e = list(k);
                ra += e > a;
                rb += e > b;
            }
        }
        __syncthreads();
        if (i < n) list(ra) = a;
        if (j < n) list(rb) = b;
        __syncthreads();
        return;
    }
    int size = 4 * NT();
    while (size < n) size <<= 1;
    for (int i = n + (int)threadIdx.x; i < size; i += NT()) list(i) = 0;
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j; j >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < size / 2; i += NT()) {
                const int lo = (i / j) * 2 * j + i % j, hi = lo + j;
                const unsigned long long a = list(lo), b = list(hi);
                if ((a < b) == ((lo & k) == 0)) {
                    list(lo) = b;
                    list(hi) = a;
                }
            }
        }
    __syncthreads();
}

__device__ void clear() {
    __syncthreads();
    for (int i = threadIdx.x; i < 4 * NB; i += NT()) digit(0, i) = 0;
    __syncthreads();
}
__device__ __forceinline__ uint64_t bin_value(int b) {
    return (uint64_t)digit(0, b) + ((uint64_t)digit(1, b) << 10) + ((uint64_t)digit(2, b) << 20) + ((uint64_t)digit(3, b) << 30);
}
// MASS: the weight high * 2^20 + low; otherwise one.
template <bool MASS>
__device__ __forceinline__ void bin_add(int b, uint32_t high, uint32_t low) {
    if (!MASS) {
        atomicAdd(&digit(0, b), 1u);
        return;
    }
    atomicAdd(&digit(0, b), low & 1023);
    atomicAdd(&digit(1, b), low >> 10);
    atomicAdd(&digit(2, b), high & 1023);
    atomicAdd(&digit(3, b), high >> 10);
}

// The first bin whose running sum reaches target, and (*before) the sum of the bins before it; -1 if none does.
__device__ int hist_find(Shared &S, uint64_t target, uint64_t *before) {
    if (threadIdx.x == 0) S.bin = -1;
    __syncthreads();
    const int per = NB / NT();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint64_t sum = 0;
    for (int i = 0; i < per; i++) sum += bin_value(threadIdx.x * per + i);
    uint64_t upto = warp_scan64(sum, lane);
    if (lane == 31) S.part[warp] = upto;
    __syncthreads();
    for (int i = 0; i < warp; i++) upto += S.part[i];
    uint64_t c = upto - sum;
    if (upto >= target && c < target) {
        for (int i = threadIdx.x * per;; i++) {
            const uint64_t v = bin_value(i);
            if (c + v >= target) {
                S.bin = i;
                S.before = c;
                break;
            }
            c += v;
        }
    }
    __syncthreads();
    *before = S.before;
    return S.bin;
}

// A histogram of the tokens above `low` at distances below `span`, by distance.
template <typename T>
struct Bins {
    float span, scale, low;
    __device__ __forceinline__ Bins(float span_, float low_) : span(span_), scale((float)NB / span_), low(low_) {}
    // The bin of a token, -1: it is not counted.  d: its distance.
    __device__ __forceinline__ int at(float f, float d) const {
        // (2^23 added and rounded towards zero leaves a whole number in the last bits, in less time than a conversion.)
        return f > low && -d < span ? min(NB - 1, (int)(__float_as_uint(__fadd_rz(-d * scale, 8388608.0f)) & 0x7fffffu)) : -1;
    }
    // Logits between which bin b's lie, and few others: its ends, moved by more than their rounding.
    __device__ __forceinline__ float2 about(const Row<T> &R, int b) const {
        const float unit = 1.0f / (scale * R.inv), far = 1e-6f * fabsf(R.m);
        if (!(unit > 1e-30f && unit < 1e30f)) return make_float2(-INFINITY, INFINITY);
        return make_float2(R.m - (float)(b + 1) * 1.00001f * unit - far, R.m - (float)b * 0.99999f * unit + far);
    }

};

// The key of the entry of a sorted list at which the running measure reaches target, and how many up to it have that key.
template <typename T, bool MASS>
__device__ uint32_t list_find(Shared &S, const Row<T> &R, int n, uint64_t target, uint64_t *ties) {
    uint64_t below = 0;
    for (int i0 = 0; i0 < n; i0 += NT()) {
        const int i = i0 + (int)threadIdx.x, warp = threadIdx.x >> 5;
        const uint64_t w = i >= n ? 0 : MASS ? R.weight(value_of(entry_key(list(i)))) : 1;
        uint64_t upto = below + warp_scan64(w, R.lane);
        if (R.lane == 31) S.part[warp] = upto - below;
        __syncthreads();
        for (int v = 0; v < NW(); v++) {
            if (v < warp) upto += S.part[v];
            below += S.part[v];
        }
        if (upto >= target && upto - w < target) {
            S.kmin = entry_key(list(i));
            S.count = i;
        }
        __syncthreads();
        if (below >= target) break;
    }
    int same = 0;
    for (int i = threadIdx.x; i <= min(S.count, n - 1); i += NT()) same += entry_key(list(i)) == S.kmin;
    if (threadIdx.x == 0) S.before = 0;
    __syncthreads();
    if (same) atomicAdd(&S.before, (unsigned long long)same);
    __syncthreads();
    *ties = S.before;
    return S.kmin;
}

// The last of the first ranks at which the running measure (tokens, or MASS:
// their weights) of the tokens in the histogram reaches target: its key, and how
// many of that key's tokens belong to the ranks (0: the measure does not reach
// target).  Not for tokens without weight.
template <typename T, bool MASS>
__device__ uint32_t select_ranks(Shared &S, const Row<T> &R, const Bins<T> &H, uint64_t target, uint64_t *ties) {
    constexpr int N = Row<T>::N;
    __syncthreads();
    uint64_t before;
    const int b = hist_find(S, target, &before);
    *ties = 0;
    if (b < 0) return 0;
    target -= before;
    // the bin's tokens: their keys' range, and the list of them if it holds them
    uint32_t lo = 0, hi = 0xffffffffu;
    for (int level = 0; level < 5; level++) {  // a range of 32 bits is down to one key after three
        const bool first = level == 0;
        __syncthreads();
        if (threadIdx.x == 0) {
            S.count = 0;
            S.kmin = 0xffffffffu;
            S.kmax = 0;
        }
        __syncthreads();
        uint32_t kmin = 0xffffffffu, kmax = 0;
        const float2 near_ = R.spike ? make_float2(-INFINITY, INFINITY) : first ? H.about(R, b) : make_float2(value_of(lo), value_of(hi));
        R.each(R.g0, R.g1, [&](const uint4 &q, int g) {
            float f[N];
            unpack<T>(q, f);
#pragma unroll
            for (int e = 0; e < N; e++) {
                if (!((f[e] >= near_.x) & (f[e] <= near_.y))) continue;
                const uint32_t k = key_of(f[e]);
                if (first ? H.at(f[e], R.dist(f[e])) != b : k < lo || k > hi) continue;
                kmin = min(kmin, k);
                kmax = max(kmax, k);
                const int i = atomicAdd(&S.count, 1);
                if (i < kList) list(i) = entry_of(k, R.index(g, e));
            }
        });
        kmin = __reduce_min_sync(0xffffffffu, kmin);
        kmax = __reduce_max_sync(0xffffffffu, kmax);
        if (R.lane == 0) {
            atomicMin(&S.kmin, kmin);
            atomicMax(&S.kmax, kmax);
        }
        __syncthreads();
        lo = S.kmin;
        hi = S.kmax;
        const int n = S.count;
        if (n <= kList || lo == hi) {
            if (lo != hi) {
                sort_list(n);
                return list_find<T, MASS>(S, R, n, target, ties);
            }
            const uint64_t w = MASS ? R.weight(value_of(hi)) : 1;
            *ties = (target + w - 1) / w;
            return hi;
        }
        // too many: a histogram of their keys, and again for the part that counts
        int shift = 0;
        while (((hi - lo) >> shift) >= NB) shift++;
        clear();
        R.each(R.g0, R.g1, [&](const uint4 &q, int) {
            float f[N];
            unpack<T>(q, f);
#pragma unroll
            for (int e = 0; e < N; e++) {
                const uint32_t k = key_of(f[e]);
                if (k >= lo && k <= hi) {
                    const uint64_t w = MASS ? R.weight(f[e]) : 0;
                    bin_add<MASS>((hi - k) >> shift, (uint32_t)(w >> 20), (uint32_t)w & 0xfffffu);
                }
            }
        });
        __syncthreads();
        const int part = hist_find(S, target, &before);
        if (part < 0) break;
        target -= before;
        hi -= (uint32_t)part << shift;
        const uint32_t width = (1u << shift) - 1;
        lo = hi - lo > width ? hi - width : lo;
    }
    return 0;
}

// floor(u * total), below total.
__device__ __forceinline__ uint64_t place(const Args &A, int64_t row, uint64_t total) {
    const double u = A.utype == ZPUCUDA_F64 ? ((const double *)A.uniform)[row] : (double)((const float *)A.uniform)[row];
    if (!(u > 0.0)) return 0;
    const double r = floor(u * (double)(int64_t)total);
    const uint64_t at = r < (double)(int64_t)total ? (uint64_t)r : total;
    return at < total ? at : total - 1;
}
__device__ __forceinline__ uint64_t top_p_edge(float p, uint64_t total) {
    const double edge = ceil((double)p * (double)(int64_t)total);
    return edge >= 1.0 ? (uint64_t)edge : 1;
}
template <typename T>
__device__ __forceinline__ void choose(const Args &A, int64_t row, const Row<T> &R, int64_t token, float f, uint64_t total) {
    A.token[row] = token;
    if (A.logprob) A.logprob[row] = R.dist(f) - logf((float)(int64_t)total / (float)kOne);
}

// floor(2^40 e), 0 <= e <= 1, as two whole numbers of 20 bits, floor(2^20 e) and floor(2^40 (e - the first / 2^20)): adding
// 8 = 2^3 to e with rounding towards zero leaves the first in the last bits of the sum, adding 2^-17 to the exact rest the
// second.
constexpr uint32_t k3 = 0x41000000u, k17 = 0x37000000u;  // 2^3, 2^-17
__device__ __forceinline__ uint2 halves(float e) {
    const float hi = __fadd_rz(e, __uint_as_float(k3)), rest = e - (hi - __uint_as_float(k3));
    return make_uint2(__float_as_uint(hi) - k3, __float_as_uint(__fadd_rz(rest, __uint_as_float(k17))) - k17);
}

// What is kept: tokens above `low` whose e^((x - max) / T) is at least `least`, and the first `ties` equal to `low`, which
// weigh wk each.
struct Kept {
    float low, least;
    uint64_t ties, wk;
    __device__ __forceinline__ float keep(float f, float e) const { return (f > low) & (e >= least) ? e : 0.0f; }
};

// The token whose running sum of kept weights by index exceeds the place.  Sums of each warp's granules first, then of
// parts of the ones that hold the place, then of those.
template <typename T>
__device__ void finish_row(Shared &S, const Row<T> &R, const Args &A, int64_t row, const Kept K) {
    constexpr int N = Row<T>::N;
    const uint64_t ties = K.ties, wk = K.wk;
    const int warp = threadIdx.x >> 5;
    auto add = [&](int a, int b, auto tied) {  // of granules a to b, to S
        const f32x2 c3 = make2(__uint_as_float(k3)), c17 = make2(__uint_as_float(k17));
        auto sub2 = [](f32x2 x, f32x2 y) { return fma2(y, make2(-1.0f), x); };
        uint64_t high = 0, low = 0;
        uint32_t t = 0;
        R.template each<2>(a, b, [&](const uint4 &q, int) {
            float f[N];
            unpack<T>(q, f);
            uint32_t h = -N * k3, l = -N * k17;
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                const f32x2 d = mul2(add2(make2(f[e], f[e + 1]), make2(-R.m)), make2(R.inv));
                const float e0 = expf(lo2(d)), e1 = expf(hi2(d));
                const f32x2 w = make2(K.keep(f[e], e0), K.keep(f[e + 1], e1));
                const f32x2 hi = add2_rz(w, c3), rest = sub2(w, sub2(hi, c3)), lo = add2_rz(rest, c17);
                h += __float_as_uint(lo2(hi)) + __float_as_uint(hi2(hi));
                l += __float_as_uint(lo2(lo)) + __float_as_uint(hi2(lo));
                if (decltype(tied)::value) t += (f[e] == K.low) + (f[e + 1] == K.low);
            }
            high += h;
            low += l;
        });
        const uint64_t s = warp_sum64((high << 20) + low);
        t = __reduce_add_sync(0xffffffffu, t);
        __syncthreads();
        if (R.lane == 0) {
            S.part[warp] = s;
            S.ties[warp] = t;
        }
        __syncthreads();
    };
    auto sums = [&](int a, int b) {
        if (ties) add(a, b, std::true_type());
        else add(a, b, std::false_type());
    };
    // the part that holds `at` once `before` and `left` ties lie before them; those are moved on.  A lane a part.
    auto find = [&](uint64_t at, uint64_t *before, uint64_t *left, uint64_t *total) {
        const uint32_t t = R.lane < NW() ? S.ties[R.lane] : 0;
        const uint64_t ties_before = warp_scan64(t, R.lane) - t, mine = *left > ties_before ? min(*left - ties_before, (uint64_t)t) : 0;
        const uint64_t w = R.lane < NW() ? S.part[R.lane] + mine * wk : 0, upto = warp_scan64(w, R.lane);
        const uint32_t over = __ballot_sync(0xffffffffu, *before + upto > at);
        const int found = over ? min(__ffs(over) - 1, NW() - 1) : NW() - 1;
        *total = __shfl_sync(0xffffffffu, upto, 31);
        *before += __shfl_sync(0xffffffffu, upto - w, found);
        const uint64_t gone = __shfl_sync(0xffffffffu, ties_before, found);
        *left -= min(*left, gone);
        return found;
    };
    sums(R.g0, R.g1);
    uint64_t before = 0, left = ties, total, unused;
    find(~0ull, &before, &left, &total);
    const uint64_t at = place(A, row, total);
    before = 0;
    left = ties;
    const int w0 = find(at, &before, &left, &unused);
    const int a = min(R.n, w0 * R.seg), b = min(R.n, a + R.seg), sub = (b - a + NW() - 1) / NW();
    sums(min(b, a + warp * sub), min(b, a + (warp + 1) * sub));
    const int w1 = find(at, &before, &left, &unused);
    if (warp != w1) return;
    // one granule a lane
    for (int g = min(b, a + w1 * sub), end = min(b, g + sub); g < end; g += 32) {
        const bool in = g + R.lane < end;
        const uint4 q = in ? R.load(g + R.lane) : make_uint4(0, 0, 0, 0);
        float f[N];
        unpack<T>(q, f);
        uint64_t s[N], sum = 0;
        uint32_t t = 0;
#pragma unroll
        for (int e = 0; e < N; e++) {
            s[e] = weigh_bits(__float_as_uint(K.keep(f[e], expf((f[e] - R.m) * R.inv))));
            t += in && f[e] == K.low;
        }
        uint32_t upto = t;  // ties up to this lane's last
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
            if (R.lane >= o) upto += v;
        }
        uint64_t rank = upto - t;
#pragma unroll
        for (int e = 0; e < N; e++) {
            if (in && f[e] == K.low && rank++ < left) s[e] = wk;
            sum += in ? s[e] : 0;
            s[e] = sum;
        }
        const uint64_t incl = warp_scan64(sum, R.lane), excl = before + incl - sum;
        const uint32_t over = __ballot_sync(0xffffffffu, before + incl > at);
        if (over) {
            if (R.lane == __ffs(over) - 1) {
                bool open = true;
#pragma unroll
                for (int e = 0; e < N; e++)
                    if (open && excl + s[e] > at) {
                        open = false;
                        choose(A, row, R, R.index(g + R.lane, e), f[e], total);
                    }
            }
            return;
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
        const uint64_t seen = __shfl_sync(0xffffffffu, upto, 31);
        left -= seen < left ? seen : left;
    }
}

// The choice among the k first ranks (k <= kQuick); false if there are too many tokens to list.
template <typename T>
__device__ bool sample_quick(Shared &S, const Row<T> &R, const Args &A, int64_t row, float mine, int k, float p, uint64_t least) {
    constexpr int N = Row<T>::N;
    const int lane = R.lane, warp = threadIdx.x >> 5;
    // the k-th largest of the threads' maxima, bit by bit; -inf is not listed
    const uint32_t key = key_of(mine);
    uint32_t bound = 0;
    for (int bit = 31; bit >= 0; bit--) {
        const uint32_t t = bound | (1u << bit);
        const int c = __syncthreads_count(key >= t);
        if (c >= k) bound = t;
        if (c == k) break;
    }
    bound = max(bound, 0x00800000u);  // the lowest finite value
    if (threadIdx.x == 0) S.count = 0;
    __syncthreads();
    const float low = value_of(bound);
    R.template each<4>(R.g0, R.g1, [&](const uint4 &q, int g) {
        if (Row<T>::largest(q) < low) return;
        float f[N];
        unpack<T>(q, f);
#pragma unroll
        for (int e = 0; e < N; e++)
            if (f[e] >= low) {
                const int i = atomicAdd(&S.count, 1);
                if (i < kList) list(i) = entry_of(key_of(f[e]), R.index(g, e));
            }
    });
    __syncthreads();
    const int n = S.count;
    if (n > kList) return false;
    sort_list(n);
    // a thread a rank
    const bool in = (int)threadIdx.x < min(k, n);
    const unsigned long long e = in ? list(threadIdx.x) : 0;
    const float f = value_of(entry_key(e));
    const uint32_t index = entry_index(e);
    uint64_t w = in ? R.weight(f) : 0;
    auto block_scan = [&](uint64_t v, uint64_t *total) {
        const uint64_t upto = warp_scan64(v, lane);
        __syncthreads();
        if (lane == 31) S.part[warp] = upto;
        __syncthreads();
        uint64_t below = 0, all = 0;
        for (int i = 0; i < NW(); i++) {
            if (i < warp) below += S.part[i];
            all += S.part[i];
        }
        *total = all;
        return below + upto;
    };
    uint64_t total;
    if (p < 1.0f) {
        const uint64_t upto = block_scan(w, &total);
        if (upto - w >= top_p_edge(p, total)) w = 0;
    }
    if (w < least) w = 0;
    block_scan(w, &total);
    const uint64_t at = place(A, row, total);
    // the running sum by index, up to this one
    S.w[threadIdx.x] = w;
    __syncthreads();
    uint64_t upto = 0;
    if (w)
        for (int j = 0; j < min(k, n); j++)
            if (entry_index(list(j)) <= index) upto += S.w[j];
    if (w && upto > at && upto - w <= at) choose(A, row, R, (int64_t)index, f, total);
    return true;
}

// 16-bit logits as whole numbers: falling logits, rising places from the largest's (0) on.  NaN has none (its place is
// past all others).  Half of all values lie within 2^-6 of zero, and few logits: those share one place, `zero`, and are
// treated one by one.
template <typename T>
struct Values {
    static constexpr uint32_t kSmall = std::is_same<T, __half>::value ? 0x2400 : 0x3c80, kMiddle = 0x8000;  // 2^-6
    uint32_t top, zero;  // the largest's order, the place of the values about zero
    static __device__ __forceinline__ uint32_t order(uint32_t raw) {  // rises with the value
        const uint32_t far = max(raw & 0x7fffu, kSmall) - kSmall;
        return raw & 0x8000u ? kMiddle - far : kMiddle + far;
    }
    __device__ __forceinline__ explicit Values(float m) {
        top = order(raw_bits(from_f<T>(m)));
        zero = top - kMiddle;
    }
    __device__ __forceinline__ uint32_t place(uint32_t raw) const { return top - order(raw); }
    // The places of a word's two values: each one's bits in rising order, then (middle - them), and of that what the small
    // ones span is taken off.
    __device__ __forceinline__ void places(uint32_t word, uint32_t (&at)[2]) const {
        const uint32_t sign = word & 0x80008000u, rising = word ^ (0x80008000u | (sign - (sign >> 15)));
        const int z = (int)zero, middle = z + (int)(0x8000u + kSmall), small = (int)(2 * kSmall + 1);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int t = middle - (int)(i ? rising >> 16 : rising & 0xffffu);
            at[i] = (uint32_t)min(max(t - small, z), t);
        }
    }
    __device__ __forceinline__ float value(uint32_t place_) const {
        const uint32_t o = top - place_, raw = o >= kMiddle ? o - kMiddle + kSmall : 0x8000u | (kMiddle - o + kSmall);
        if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(raw << 16);
        else return __half2float(__ushort_as_half((unsigned short)raw));
    }
};

// The kept ranks of 16-bit logits (k > 0 or p < 1) from counts of each value at `n` places from the largest on (what lies
// past them has no weight): the key of the last, 0: all, and in *ties how many of that key.  False: the ranks end among
// more values about zero than are listed, or top_k's do and top_p follows.
template <typename T>
__device__ bool select_values(Shared &S, const Row<T> &R, int n, int64_t k, float p, uint32_t *key, uint64_t *ties_) {
    static_assert(sizeof(T) == 2, "16-bit logits");
    uint32_t *table = sample_smem;
    const int lane = R.lane, warp = threadIdx.x >> 5;
    const Values<T> O(R.m);
    auto raw_of = [](const uint4 &q, int e) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
        return e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu;
    };
    auto float_of = [](uint32_t raw) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(raw << 16);
        else return __half2float(__ushort_as_half((unsigned short)raw));
    };
    // The kept ranks: places below `last`, and the first `ties` tokens at it.
    uint32_t last = (uint32_t)n;
    uint64_t ties = 0;
    for (int i = threadIdx.x; i < n; i += NT()) table[i] = 0;
    __syncthreads();
    unsigned short *near_ = (unsigned short *)(sample_smem + kPlaces);
    if (threadIdx.x == 0) S.count = 0;
    __syncthreads();
    const uint32_t zero = O.zero < (uint32_t)n ? O.zero : 0xffffffffu;
    R.each(R.g0, R.g1, [&](const uint4 &q, int) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            uint32_t at[2];
            O.places(w[e], at);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                atomicAdd(&table[min(at[i], (uint32_t)(n + lane))], 1u);  // past the places: not looked at
                if (at[i] == zero) {
                    const int to = atomicAdd(&S.count, 1);
                    if (to < kNear) near_[to] = (unsigned short)(i ? w[e] >> 16 : w[e]);
                }
            }
        }
    });
    __syncthreads();
    uint64_t about = 0;  // the weight of the values about zero
    const int nears = S.count;
    if (p >= 1.0f) {
    } else if (nears <= kNear) {
        for (int i = threadIdx.x; i < nears; i += NT()) about += R.weight(float_of(near_[i]));
    } else {
        R.each(R.g0, R.g1, [&](const uint4 &q, int) {
            for (int e = 0; e < 8; e++) {
                const uint32_t raw = raw_of(q, e);
                if (O.place(raw) == zero) about += R.weight(float_of(raw));
            }
        });
    }
    about = warp_sum64(about);
    if (lane == 0) S.w[warp] = about;
    __syncthreads();
    about = 0;
    for (int i = 0; i < NW(); i++) about += S.w[i];
    // A warp has a run of places.  What they measure, and the place at which the running measure reaches target, with
    // what is left of the target there; all threads get both (n: it does not reach target).
    const int per = (n + NT() - 1) / NT() * 32, b0 = min(n, warp * per), b1 = min(n, b0 + per);
    auto reach = [&](auto measure, auto target_of, uint64_t *rest) {
        uint64_t c = 0;
        for (int i = b0 + lane; i < b1; i += 32) c += measure(i);
        c = warp_sum64(c);
        __syncthreads();
        if (lane == 0) S.part[warp] = c;
        if (threadIdx.x == 0) S.bin = n;
        __syncthreads();
        uint64_t before = 0, total = 0;
        for (int i = 0; i < NW(); i++) {
            before += i < warp ? S.part[i] : 0;
            total += S.part[i];
        }
        const uint64_t target = target_of(total);
        if (before < target && before + c >= target) {  // this warp's, a run of places a lane
            const int run = (b1 - b0 + 31) / 32, r0 = min(b1, b0 + lane * run), r1 = min(b1, r0 + run);
            uint64_t v = 0;
            for (int i = r0; i < r1; i++) v += measure(i);
            uint64_t s = before + warp_scan64(v, lane) - v;
            if (s < target && s + v >= target)
                for (int i = r0; i < r1; i++) {
                    const uint64_t m = measure(i);
                    if (s + m >= target) {
                        S.bin = i;
                        S.before = target - s;
                        break;
                    }
                    s += m;
                }
        }
        __syncthreads();
        *rest = S.before;
        return (uint32_t)S.bin;
    };
    if (k > 0) {
        last = reach([&](int i) -> uint64_t { return table[i]; }, [&](uint64_t) { return (uint64_t)k; }, &ties);
        if (last == (uint32_t)n) ties = 0;
        if (last == O.zero && p < 1.0f) return false;
    }
    if (p < 1.0f) {
        const uint32_t end = last;
        const uint64_t some = ties;  // of the end's tokens, those that top_k leaves
        uint64_t rest;
        last = reach(
            [&](int i) -> uint64_t {
                const uint64_t m = (uint32_t)i < end ? table[i] : (uint32_t)i == end ? some : 0;
                return (uint32_t)i == O.zero ? (m ? about : 0) : m ? m * R.weight(O.value(i)) : 0;
            },
            [&](uint64_t total) { return top_p_edge(p, total); }, &rest);
        if (last == (uint32_t)n) return false;
        if (last != O.zero) {
            const uint64_t w = R.weight(O.value(last));
            rest = (rest + w - 1) / w;
        }
        ties = rest;
    }
    if (last == zero) {  // its tokens in order, up to the rest of the target
        if (nears > kNear) return false;
        for (int i = threadIdx.x; i < nears; i += NT()) list(i) = entry_of(key_of(float_of(near_[i])), i);
        sort_list(nears);
        *key = p < 1.0f ? list_find<T, true>(S, R, nears, ties, ties_) : list_find<T, false>(S, R, nears, ties, ties_);
        return true;
    }
    __syncthreads();
    *key = last < (uint32_t)n ? key_of(O.value(last)) : 0;
    *ties_ = *key ? ties : 0;
    return true;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const T *logits, int64_t ld, const Args A) {
    constexpr int N = Row<T>::N;
    __shared__ Shared S;
    const int64_t row = blockIdx.x, V = A.vocab;
    const int warp = threadIdx.x >> 5;
    Row<T> R;
    R.vocab = V;
    R.lane = threadIdx.x & 31;
    const T *x = logits + row * ld;
    R.skew = (int)(((uintptr_t)x & 15) / sizeof(T));
    R.x = x - R.skew;
    R.n = (int)((R.skew + V + N - 1) / N);
    R.seg = (R.n + NW() - 1) / NW();
    R.g0 = min(R.n, warp * R.seg);
    R.g1 = min(R.n, R.g0 + R.seg);

    R.first = R.skew ? 1 : 0;
    R.last = (R.skew + V) % N ? R.n - 1 : R.n;
    R.edge = S.edge;
    if (threadIdx.x == 0 && R.first) S.edge[0] = R.load_edge(0);
    if (threadIdx.x == 1 && R.last < R.n && R.n > R.first) S.edge[1] = R.load_edge(R.n - 1);
    __syncthreads();

    float mine = -INFINITY;
    int at = 0;  // the first granule that has it
    R.template each<4>(R.g0, R.g1, [&](const uint4 &q, int g) {
        const float t = Row<T>::largest(q);
        if (t > mine || (t == mine && g < at)) {
            mine = t;
            at = g;
        }
    });
    float m = mine;
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (R.lane == 0) S.fmax_[warp] = m;
    __syncthreads();
    for (int w = 0; w < NW(); w++) m = fmaxf(m, S.fmax_[w]);
    if (m == -INFINITY) {
        if (threadIdx.x == 0) {
            A.token[row] = -1;
            if (A.logprob) A.logprob[row] = -INFINITY;
        }
        return;
    }
    const float temp = A.temperature ? A.temperature[row] : 1.0f;
    R.m = m;
    R.inv = temp > 0.0f ? 1.0f / temp : 0.0f;
    R.spike = isinf(m) || isinf(R.inv);
    const float p = A.top_p ? A.top_p[row] : 1.0f, mp = A.min_p ? A.min_p[row] : 0.0f;
    uint64_t least = 0;
    if (mp > 0.0f) least = mp < 1.0f ? (uint64_t)ceil((double)mp * (double)kOne) : kOne;

    // The kept ranks: keys above `key`, and the first `ties` tokens of that key.
    uint32_t key = 0;
    uint64_t ties = 0;
    if (!(temp > 0.0f)) {  // the first of the largest
        if (threadIdx.x == 0) S.count = R.n;
        __syncthreads();
        if (mine == m) atomicMin(&S.count, at);
        __syncthreads();
        if (mine == m && at == S.count) {
            float f[N];
            unpack<T>(R.load(at), f);
            bool open = true;
#pragma unroll
            for (int e = 0; e < N; e++)
                if (open && f[e] == m) {
                    open = false;
                    choose(A, row, R, R.index(at, e), f[e], kOne);
                }
        }
        return;
    }
    bool known = false;
    {
        const int64_t k = A.top_k ? A.top_k[row] : 0;
        if (k > 0 && k <= kQuick && k < V && sample_quick(S, R, A, row, mine, (int)k, p, least)) return;
        if constexpr (sizeof(T) == 2) {
            // places down to the last value with weight (a little lower does no harm), if the table holds them
            const float lowest = R.spike ? m : fmaxf(m - kSpan / R.inv, -3.0e38f);
            const int n = (int)Values<T>(m).place(raw_bits(from_f<T>(lowest))) + 2;  // lowest is rounded to nearest: kSpan has room
            if ((p < 1.0f || (k > 0 && k < V)) && n + 32 <= A.places)
                known = select_values(S, R, n, k < V ? k : 0, p, &key, &ties);
        }
        if (!known && k > 0 && k < V) {
            const Bins<T> H(kSpan, -INFINITY);
            clear();
            R.each(R.g0, R.g1, [&](const uint4 &q, int) {
                float f[N];
                unpack<T>(q, f);
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const int b = H.at(f[e], R.dist(f[e]));
                    if (b >= 0) bin_add<false>(b, 0, 0);
                }
            });
            key = select_ranks<T, false>(S, R, H, (uint64_t)k, &ties);
        }
        if (!known && p < 1.0f) {
            // Tokens that, all together, weigh less than what the set leaves out are not in it: with the whole weight at
            // least `sure` (of the threads' largest tokens; with a top_k set, of the largest token), those lighter than
            // (1 - p) sure / vocab are left out of the histogram (a distance a little larger stands for that weight).
            const float low = key ? value_of(key) : -INFINITY;
            uint64_t sure = mine > -INFINITY && !key ? R.weight(mine) : 0;
            sure = warp_sum64(sure);
            __syncthreads();
            if (R.lane == 0) S.part[warp] = sure;
            clear();
            sure = 0;
            for (int i = 0; i < NW(); i++) sure += S.part[i];
            if (sure < kOne) sure = kOne;
            const float light = (1.0f - p) * (float)sure / (float)kOne / (float)V;
            const float span = p > 0.0f && light > 0.0f ? fminf(kSpan, fmaxf(1e-3f, 1e-3f - logf(light))) : kSpan;
            const Bins<T> H(span, low);
            uint64_t sum = 0;
            R.each(R.g0, R.g1, [&](const uint4 &q, int) {
                float f[N];
                unpack<T>(q, f);
                uint32_t high = 0, rest = 0;  // sums of the weights' two halves
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const float d = R.dist(f[e]), p = f[e] > low ? R.spike ? (f[e] == m ? 1.0f : 0.0f) : expf(d) : 0.0f;
                    const uint2 w = halves(p);
                    high += w.x;
                    rest += w.y;
                    const int b = H.at(f[e], d);
                    if (b >= 0) bin_add<true>(b, w.x, w.y);
                }
                sum += ((uint64_t)high << 20) + rest;
            });
            sum = warp_sum64(sum);
            __syncthreads();
            if (R.lane == 0) S.part[warp] = sum;
            __syncthreads();
            uint64_t above = 0;
            for (int i = 0; i < NW(); i++) above += S.part[i];
            __syncthreads();
            const uint64_t wk = key ? R.weight(value_of(key)) : 0, target = top_p_edge(p, above + ties * wk);
            if (above >= target) {
                key = select_ranks<T, true>(S, R, H, target, &ties);
            } else {
                const uint64_t need = (target - above + wk - 1) / wk;  // wk > 0: the total is above `above`
                ties = need < ties ? need : ties;
            }
        }
    }

    if (R.spike && key != key_of(m)) {  // the largest alone have weight
        key = key_of(m);
        ties = (uint64_t)V;
    }
    Kept K = {key ? value_of(key) : -INFINITY, __ull2float_ru(least) / (float)kOne, key ? ties : 0, key ? R.weight(value_of(key)) : 0};
    if (K.wk < least) K.wk = 0;
    finish_row(S, R, A, row, K);
}

template <typename T>
int launch_sample(const T *logits, int64_t ld, const Args &A, int64_t rows, cudaStream_t s) {
    auto f = sample_kernel<T>;
    const size_t smem = sizeof(T) == 2 ? kPlaces * sizeof(uint32_t) + kNear * sizeof(short) : kSmem;
    static int cache[64] = {0};
    if (!blocks_per_sm(f, kThreads, smem, smem, cache)) return cuda_fail(cudaGetLastError(), "sample: occupancy");
    const int threads = rows <= num_sms() ? kThreads : kThreads / 2;
    f<<<(unsigned)rows, threads, smem, s>>>(logits, ld, A);
    ZC_LAUNCHED("sample_kernel");
    return ZPUCUDA_OK;
}

}  // namespace
}  // namespace zc

using namespace zc;

extern "C" int zpucuda_sample(int dtype, const void *d_logits, int64_t ld, int utype, const void *d_uniform,
                              const float *d_temperature, const int32_t *d_top_k, const float *d_top_p,
                              const float *d_min_p, int64_t *d_token, float *d_logprob, int64_t rows, int64_t vocab,
                              void *stream) {
    if (rows < 0 || vocab < 1) return set_error(ZPUCUDA_ERR_INVALID_SHAPE, "sample: rows >= 0 and vocab >= 1 are wanted");
    if (vocab > kMaxVocab) return set_error(ZPUCUDA_ERR_NOT_SUPPORTED, "sample: 2^22 tokens or more");
    if (rows > 0x7fffffff) return set_error(ZPUCUDA_ERR_NOT_SUPPORTED, "sample: more than 2^31 - 1 rows");
    ZC_TRY(check_matrix("sample", "logits", d_logits, dtype, ld, rows, vocab));
    if (utype != ZPUCUDA_F32 && utype != ZPUCUDA_F64) return set_error(ZPUCUDA_ERR_NOT_SUPPORTED, "sample: uniform is not f32 or f64");
    ZC_TRY(check_vectors("sample", utype == ZPUCUDA_F64 ? 8 : 4, {{"uniform", d_uniform}}));
    ZC_TRY(check_vectors("sample", 4, {{"temperature", d_temperature}, {"top_k", d_top_k}, {"top_p", d_top_p}, {"min_p", d_min_p}, {"logprob", d_logprob}}));
    ZC_TRY(check_vectors("sample", 8, {{"token", d_token}}));
    if (rows == 0) return ZPUCUDA_OK;
    if (!d_uniform || !d_token) return set_error(ZPUCUDA_ERR_INVALID_ARGUMENT, "sample: uniform or token: null pointer");
    const Args A = {d_uniform, utype, d_temperature, d_top_k, d_top_p, d_min_p, d_token, d_logprob, vocab, kPlaces};
    cudaStream_t s = resolve_stream(stream);
    ZC_HEAD_TYPE(dtype, T, return launch_sample((const T *)d_logits, ld, A, rows, s));
}
