// What the serving operators (tt_q4.hip, tt_kv_append.hip, tt_kv_attention.hip)
// share: element types, 8-bit codes, and the checks of a cache.
#pragma once

#include "tt_common.hpp"

namespace tt {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kFp8Max = 448.f;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__bf16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(_Float16 x) { return (float)x; }

// One e4m3 code as a float.
__device__ __forceinline__ float fp8_value(uint8_t c) { return __builtin_amdgcn_cvt_f32_fp8((int)c, 0); }

// Two floats as e4m3 codes (low byte first): nearest even, saturated, NaN kept.
__device__ __forceinline__ uint32_t fp8_pair(float a, float b) {
    a = a > kFp8Max ? kFp8Max : (a < -kFp8Max ? -kFp8Max : a);
    b = b > kFp8Max ? kFp8Max : (b < -kFp8Max ? -kFp8Max : b);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu;
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    bf16x2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
}

__device__ __forceinline__ float bf16_of(uint32_t pair, int i) {
    return __uint_as_float(i ? pair & 0xffff0000u : pair << 16);
}

// Eight floats as N bfloat16 parts whose sum is the float to 8 N bits.
template <int N>
__device__ __forceinline__ void split8(const float* x, u32x4* out) {
    float rest[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) rest[i] = x[i];
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            out[n][i] = pack_bf16(rest[2 * i], rest[2 * i + 1]);
            if (n + 1 < N) {
                rest[2 * i] -= bf16_of(out[n][i], 0);
                rest[2 * i + 1] -= bf16_of(out[n][i], 1);
            }
        }
    }
}

// Maximum and sum over the four lanes that share a column of an MFMA's result
// (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float column_max(float x) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float column_sum(float x) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Codes of one cache row: dim rounded up to a multiple of 64.
inline int64_t kv_width(int64_t dim) { return (dim + 63) / 64 * 64; }

inline bool serving_dtype(int64_t dtype) { return dtype == TT_F32 || dtype == TT_BF16 || dtype == TT_F16; }

// The checks every call on a cache makes; TT_OK or a status with its message set.
inline int check_cache(const char* who, const tt_kv_cache& c) {
    if (c.pages < 0 || c.heads < 1 || c.page < 16 || c.page % 16 || c.page > 65536 || c.dim < 1)
        return set_error(TT_INVALID, "%s: cache of %lld pages, %lld heads, %lld tokens a page, dim %lld", who,
                         (long long)c.pages, (long long)c.heads, (long long)c.page, (long long)c.dim);
    if (c.dim > 256)
        return set_error(TT_UNSUPPORTED, "%s: head size %lld (at most 256)", who, (long long)c.dim);
    if (c.pages > 0 && (!c.k || !c.v || !c.k_scale || !c.v_scale))
        return set_error(TT_INVALID, "%s: NULL cache pointer", who);
    if (((uintptr_t)c.k | (uintptr_t)c.v) % 16)
        return set_error(TT_INVALID, "%s: cache pointers are not 16-byte aligned", who);
    return TT_OK;
}

}  // namespace tt
