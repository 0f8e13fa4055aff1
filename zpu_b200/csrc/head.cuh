// What the language-model head's kernels share (layernorm.cu, distill.cu,
// int8.cu, sample.cu): their element types, conversions, block sums and
// argument checks.  These operators take f32, f16 and bf16 (ZPUCUDA_BF16);
// every sum is held in f32 or wider, and a result is rounded to its type
// once, when it is stored.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include <initializer_list>
#include <type_traits>
#include <utility>

#include "common.cuh"
#include "head_rules.h"

namespace zc {

inline int elem_bytes(int dt) { return dt == ZPUCUDA_F32 ? 4 : 2; }
inline bool is_head_type(int dt) { return dt == ZPUCUDA_F32 || dt == ZPUCUDA_F16 || dt == ZPUCUDA_BF16; }
inline bool aligned_to(const void *p, size_t n) { return ((uintptr_t)p % n) == 0; }

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Element i of a buffer of one of the head's types, as f32.
__device__ __forceinline__ float load_f(const void *p, int dt, int64_t i) {
    if (dt == ZPUCUDA_F32) return ((const float *)p)[i];
    if (dt == ZPUCUDA_F16) return __half2float(((const __half *)p)[i]);
    return __bfloat162float(((const __nv_bfloat16 *)p)[i]);
}
__device__ __forceinline__ void store_f(void *p, int dt, int64_t i, float v) {
    if (dt == ZPUCUDA_F32) ((float *)p)[i] = v;
    else if (dt == ZPUCUDA_F16) ((__half *)p)[i] = __float2half_rn(v);
    else ((__nv_bfloat16 *)p)[i] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// The larger of two values; a NaN among them stays.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// ---- rows in pieces of 16 bytes
// Piece i of a row holds its elements i * N .. i * N + N - 1 (N = 16 / the
// element's size), wherever the row starts: an address that is no multiple of
// 16 costs a second load and some shifts, not another order of a sum, so a
// result does not depend on the alignment.  Nothing outside the row is touched,
// except that RowRing reads the aligned 16 bytes in which a row begins, as far as
// they lie in its matrix, and drops what comes before the row.

template <typename T>
constexpr int kPiece = 16 / (int)sizeof(T);

// Two f32 values in one register pair: sm_100 adds and multiplies both with one
// instruction, each rounded as by itself.
struct f32x2 {
    unsigned long long v;
};
__device__ __forceinline__ f32x2 make2(float lo, float hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ f32x2 make2(float x) { return make2(x, x); }
__device__ __forceinline__ float lo2(f32x2 a) { return __uint_as_float((uint32_t)a.v); }
__device__ __forceinline__ float hi2(f32x2 a) { return __uint_as_float((uint32_t)(a.v >> 32)); }
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ f32x2 add2_rz(f32x2 a, f32x2 b) {  // rounded towards zero
    f32x2 r;
    asm("add.rz.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4 &q, float (&f)[kPiece<T>]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                f[2 * i] = __uint_as_float(w[i] << 16);
                f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
                const __half2 h = *(const __half2 *)&w[i];
                f[2 * i] = __low2float(h);
                f[2 * i + 1] = __high2float(h);
            }
        }
    }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float (&f)[kPiece<T>]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) {
            w[i] = __float_as_uint(f[i]);
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *(const uint32_t *)&h;
        } else {
            const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *(const uint32_t *)&h;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T>
__device__ __forceinline__ void unpack2(const uint4 &q, f32x2 (&f)[kPiece<T> / 2]) {
    float x[kPiece<T>];
    unpack<T>(q, x);
#pragma unroll
    for (int i = 0; i < kPiece<T> / 2; i++) f[i] = make2(x[2 * i], x[2 * i + 1]);
}
template <typename T>
__device__ __forceinline__ uint4 pack2(const f32x2 (&f)[kPiece<T> / 2]) {
    float x[kPiece<T>];
#pragma unroll
    for (int i = 0; i < kPiece<T> / 2; i++) {
        x[2 * i] = lo2(f[i]);
        x[2 * i + 1] = hi2(f[i]);
    }
    return pack<T>(x);
}

// Bytes s .. s + 15 of the 32 bytes lo, hi (0 <= s < 16).
__device__ __forceinline__ uint4 bytes_from(const uint4 &lo, const uint4 &hi, uint32_t s) {
    uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int i = 0; i < 6; i++) w[i] = (s & 8) ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; i++) w[i] = (s & 4) ? w[i + 1] : w[i];
    const uint32_t b = (s & 3) * 8;
    return make_uint4(__funnelshift_r(w[0], w[1], b), __funnelshift_r(w[1], w[2], b), __funnelshift_r(w[2], w[3], b),
                      __funnelshift_r(w[3], w[4], b));
}

template <typename T>
__device__ __forceinline__ uint32_t raw_bits(T x) {
    if constexpr (sizeof(T) == 4) return *(const uint32_t *)&x;
    else return *(const uint16_t *)&x;
}

// Piece i of the row (its elements past n are 0).
template <typename T>
__device__ __forceinline__ uint4 load_piece(const T *row, int64_t i, int64_t n) {
    constexpr int N = kPiece<T>;
    const T *p = row + i * N;
    const uint32_t s = (uint32_t)(uintptr_t)p & 15;
    if ((i + 1) * N <= n) {
        if (s == 0) return *(const uint4 *)p;
        const uint4 *q = (const uint4 *)((uintptr_t)p & ~(uintptr_t)15);
        if (i > 0 && (const T *)(q + 2) <= row + n) return bytes_from(q[0], q[1], s);
    }
    uint32_t w[4] = {};
#pragma unroll
    for (int e = 0; e < N; e++)
        if (i * N + e < n) w[e * (int)sizeof(T) / 4] |= raw_bits(p[e]) << (e * (int)sizeof(T) % 4 * 8);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T>
__device__ __forceinline__ void store_elements(T *p, const uint4 &q, int from, int to) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < kPiece<T>; e++)
        if (e >= from && e < to) {
            if constexpr (sizeof(T) == 4) ((uint32_t *)p)[e] = w[e];
            else ((uint16_t *)p)[e] = (uint16_t)(w[e / 2] >> (e % 2 * 16));
        }
}

// Stores piece i of the row (its elements below n), for a whole warp at a time:
// lane l has piece i0 + l, and those past the row's end store nothing.  Where the
// row starts off a 16-byte boundary, each lane stores the 16 aligned bytes that
// hold its neighbour's end and its own beginning.
template <typename T>
__device__ __forceinline__ void store_piece(T *row, int64_t i, int64_t n, const uint4 &v) {
    constexpr int N = kPiece<T>;
    T *p = row + i * N;
    const uint32_t s = (uint32_t)(uintptr_t)p & 15;
    const int64_t rest = n - i * N;
    const int have = rest >= N ? N : rest > 0 ? (int)rest : 0;  // elements of this piece
    if (s == 0) {
        if (have == N) *(uint4 *)p = v;
        else store_elements(p, v, 0, have);
        return;
    }
    uint4 before;
    before.x = __shfl_up_sync(0xffffffffu, v.x, 1);
    before.y = __shfl_up_sync(0xffffffffu, v.y, 1);
    before.z = __shfl_up_sync(0xffffffffu, v.z, 1);
    before.w = __shfl_up_sync(0xffffffffu, v.w, 1);
    const int lane = threadIdx.x & 31;
    const int head = (int)(16 - s) / (int)sizeof(T);  // elements up to the boundary
    if (lane > 0 && have >= head) {
        *(uint4 *)((uintptr_t)p & ~(uintptr_t)15) = bytes_from(before, v, 16 - s);
    } else {
        // the neighbour's end, unless it is another warp's, and what there is of the beginning
        if (lane > 0 && rest + N > head) store_elements(p - N, before, head, rest + N < N ? (int)rest + N : N);
        store_elements(p, v, 0, have < head ? have : head);
    }
    if (lane == 31) store_elements(p, v, head, have);
}

// Stores a warp's run of pieces: lane l has pieces i = i0 + l, i + 32 and so on.  As
// above, but single elements are stored at the run's ends and the row's alone.
template <typename T, int NV>
__device__ __forceinline__ void store_run(T *row, int i, int n, const uint4 (&v)[NV]) {
    constexpr int N = kPiece<T>;
    const uint32_t s = (uint32_t)(uintptr_t)row & 15;
    const int lane = threadIdx.x & 31, head = (int)(16 - s) / (int)sizeof(T);  // elements up to the boundary
    uint4 carry = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < NV; j++) {
        T *p = row + (i + 32 * j) * N;
        const int rest = n - (i + 32 * j) * N, have = rest >= N ? N : rest > 0 ? rest : 0;
        if (s == 0) {
            if (have == N) *(uint4 *)p = v[j];
            else if (have) store_elements(p, v[j], 0, have);
            continue;
        }
        uint4 turn;  // lane 0: what goes before its next piece
        turn.x = __shfl_sync(0xffffffffu, v[j].x, (lane + 31) & 31);
        turn.y = __shfl_sync(0xffffffffu, v[j].y, (lane + 31) & 31);
        turn.z = __shfl_sync(0xffffffffu, v[j].z, (lane + 31) & 31);
        turn.w = __shfl_sync(0xffffffffu, v[j].w, (lane + 31) & 31);
        const uint4 before = lane ? turn : carry;
        carry = turn;
        const bool joined = lane > 0 || j > 0;
        if (joined && have >= head) {
            *(uint4 *)((uintptr_t)p & ~(uintptr_t)15) = bytes_from(before, v[j], 16 - s);
        } else if (joined ? rest + N > head : have > 0) {
            if (joined) store_elements(p - N, before, head, rest + N < N ? rest + N : N);
            store_elements(p, v[j], 0, have < head ? have : head);
        }
        if (j == NV - 1 && lane == 31 && have > head) store_elements(p, v[j], head, have);
        __syncwarp();
    }
}

// A ring of D rows' pieces in shared memory, filled by asynchronous copies: a warp
// has a run of 32 * NV pieces of ROWS rows (tensors) a slot, lane l the pieces
// p = p0 + l, p + 32 and so on, and no other warp reads them.  Bytes in flight cost
// no registers this way.  EVEN: rows start on 16-byte boundaries and hold whole
// pieces.
template <typename T, int NV, int ROWS, int D, bool EVEN>
struct RowRing {
    static constexpr int kWarp = D * ROWS * (NV * 32 + 1);  // uint4 a warp: the run's, and the next 16 bytes
    uint4 *base;
    int lane, p;

    __device__ __forceinline__ RowRing(uint4 *smem, int p_)
        : base(smem + (threadIdx.x >> 5) * kWarp), lane(threadIdx.x & 31), p(p_) {}
    __device__ __forceinline__ uint4 *at(int slot, int r, int j) const { return base + (slot * ROWS + r) * (NV * 32 + 1) + j * 32; }

    static __device__ __forceinline__ void copy(uint4 *dst, const uint8_t *src, int size) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)),
                     "l"(src), "r"(size)
                     : "memory");
    }
    // The aligned 16 bytes that hold the row's pieces, clipped at its end and at the
    // matrix's beginning (`before`: elements of the matrix before the row).
    __device__ __forceinline__ void issue(int slot, int r, const T *row, int64_t n, int64_t before) const {
        const uint32_t s = EVEN ? 0 : (uint32_t)(uintptr_t)row & 15;
        const uint8_t *from = (const uint8_t *)row - s;
        const int end = (int)s + (int)n * (int)sizeof(T);
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int b = (p + j * 32) * 16;
            if (b >= end) continue;
            uint4 *dst = at(slot, r, j);
            if constexpr (EVEN) {
                copy(dst + lane, from + b, 16);
                continue;
            }
            if (b == 0 && begins_outside(before, (int)(s / sizeof(T)))) {
                T *e = (T *)(dst + lane);  // 0 outside the row, as the copies leave it
                for (int i = 0, at = -(int)(s / sizeof(T)); i < kPiece<T>; i++, at++) e[i] = at >= 0 && at < n ? row[at] : from_f<T>(0.0f);
            } else {
                copy(dst + lane, from + b, end - b < 16 ? end - b : 16);
            }
            if (j == NV - 1 && s && lane == 31 && b + 16 < end) copy(dst + 32, from + b + 16, end - b < 32 ? end - b - 16 : 16);
        }
    }
    static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
    // Until all but the last D - 1 groups have landed, for the whole warp.
    static __device__ __forceinline__ void wait() {
        asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory");
        __syncwarp();
    }
    // Piece t + j * TPR, 0 past the row's end.
    __device__ __forceinline__ uint4 read(int slot, int r, int j, const T *row, int64_t n) const {
        const uint32_t s = EVEN ? 0 : (uint32_t)(uintptr_t)row & 15;
        const int b = (p + j * 32) * 16, end = (int)s + (int)n * (int)sizeof(T);
        const uint4 *src = at(slot, r, j) + lane, none = make_uint4(0, 0, 0, 0);
        const uint4 lo = b < end ? src[0] : none;
        if (EVEN || s == 0) return lo;
        return bytes_from(lo, b + 16 < end ? src[1] : none, s);
    }
};

// Calls F<type> for one of the head's element types.
#define ZC_HEAD_TYPE(dt, T, ...)                                   \
    do {                                                           \
        if ((dt) == ZPUCUDA_F32) {                                 \
            using T = float;                                       \
            __VA_ARGS__;                                           \
        } else if ((dt) == ZPUCUDA_F16) {                          \
            using T = __half;                                      \
            __VA_ARGS__;                                           \
        } else {                                                   \
            using T = __nv_bfloat16;                               \
            __VA_ARGS__;                                           \
        }                                                          \
    } while (0)

// A [rows, cols] matrix argument `name` of `who`, of type dt and row pitch ld.
inline int check_matrix(const char *who, const char *name, const void *p, int dt, int64_t ld, int64_t rows,
                        int64_t cols) {
    const auto fail = [&](int st, const char *what) { return set_error(st, std::string(who) + ": " + name + ": " + what); };
    if (!is_head_type(dt)) return fail(ZPUCUDA_ERR_NOT_SUPPORTED, "the type is not f32, f16 or bf16");
    if (ld < cols) return fail(ZPUCUDA_ERR_INVALID_SHAPE, "the row pitch is below the row's length");
    if (rows > 0 && cols > 0 && !p) return fail(ZPUCUDA_ERR_INVALID_ARGUMENT, "null pointer");
    if (!aligned_to(p, elem_bytes(dt))) return fail(ZPUCUDA_ERR_INVALID_ARGUMENT, "not aligned to its elements");
    return ZPUCUDA_OK;
}
// Vector arguments `names` of `who`, any of them null, of elements of `bytes` each.
inline int check_vectors(const char *who, size_t bytes, std::initializer_list<std::pair<const char *, const void *>> vectors) {
    for (const auto &v : vectors)
        if (!aligned_to(v.second, bytes))
            return set_error(ZPUCUDA_ERR_INVALID_ARGUMENT, std::string(who) + ": " + v.first + ": not aligned to its elements");
    return ZPUCUDA_OK;
}
inline int head_error(int st, const char *who, const char *what) { return set_error(st, std::string(who) + ": " + what); }
// Blocks of f that an SM holds at once with `smem` bytes each (looked up once a
// device, for the first size asked for), after allowing it `allow`.
template <typename F>
int blocks_per_sm(F f, int block, size_t smem, size_t allow, int *cache) {
    const int dev = current_device();
    if (dev >= 0 && dev < 64 && cache[dev]) return cache[dev];
    int n = 0;
    if (cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)allow) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, f, block, smem) != cudaSuccess || n < 1)
        return 0;
    if (dev >= 0 && dev < 64) cache[dev] = n;
    return n;
}

#define ZC_TRY(call)                  \
    do {                              \
        const int st_ = (call);       \
        if (st_) return st_;          \
    } while (0)

}  // namespace zc
