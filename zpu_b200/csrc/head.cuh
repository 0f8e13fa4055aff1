// What the language-model head's kernels share (layernorm.cu, distill.cu,
// int8.cu, sample.cu): their element types, conversions, block sums and
// argument checks.  These operators take f32, f16 and bf16 (ZPUCUDA_BF16);
// every sum is held in f32 or wider, and a result is rounded to its type
// once, when it is stored.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"

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
inline int head_error(int st, const char *who, const char *what) { return set_error(st, std::string(who) + ": " + what); }
#define ZC_TRY(call)                  \
    do {                              \
        const int st_ = (call);       \
        if (st_) return st_;          \
    } while (0)

}  // namespace zc
