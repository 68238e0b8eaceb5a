// What the 8-bit chain's kernels (tt_fp8_rows.hip, tt_fp8.hip) share: rows in
// 8 bits, their layout and their rounding.
//
// A row of `dim` elements is held as e4m3 codes, fp8_width(dim) of them with
// zeros past dim, and one power of two for each block of 128, as the byte e +
// 127 (e8m0), fp8_scales(dim) of them with zeros past the blocks. The scaled
// matrix instructions take both as they are.
#pragma once

#include <type_traits>

#include "tt_serving.hpp"

namespace tt {

inline __host__ __device__ int64_t fp8_blocks(int64_t dim) { return (dim + 127) / 128; }
inline __host__ __device__ int64_t fp8_width(int64_t dim) { return fp8_blocks(dim) * 128; }
inline __host__ __device__ int64_t fp8_scales(int64_t dim) { return (fp8_blocks(dim) + 3) / 4 * 4; }

// Lanes that a row takes in tt_fp8_quantize, eight elements each (or 256 a piece of
// 2048 elements), and its workgroups of 256.
inline int fp8_quantize_lanes(int64_t dim) {
    const int64_t blocks = fp8_blocks(dim);
    return blocks <= 1 ? 16 : blocks <= 2 ? 32 : blocks <= 4 ? 64 : blocks <= 8 ? 128 : 256;
}
inline int64_t fp8_quantize_grid(int64_t rows, int64_t dim) {
    const int each = 256 / fp8_quantize_lanes(dim);
    return each > 1 ? (rows + each - 1) / each : rows * ((dim + 2047) / 2048);
}

// The e8m0 byte of a block whose largest finite magnitude is amax: the
// smallest e >= -127 with amax <= 448 * 2^e. 448 is 1.75 * 2^8, so that e is
// amax's exponent less 8, and one more where its fraction passes 1.75.
__device__ __forceinline__ uint32_t fp8_scale_byte(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);
    return e > 0 ? (uint32_t)e : 0u;
}

// 2^-e of that byte (its e is at most 120).
__device__ __forceinline__ float fp8_scale_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

__device__ __forceinline__ float finite_magnitude(float x) {
    x = fabsf(x);
    return x <= 3.402823466e38f ? x : 0.f;
}

// Maximum over 16 neighbouring lanes (those of one block, 8 elements each).
__device__ __forceinline__ float max_of_16(float x) {
    x = fmaxf(x, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x128, 0xf, 0xf, true)));  // row_ror
    x = fmaxf(x, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x124, 0xf, 0xf, true)));
    x = fmaxf(x, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x122, 0xf, 0xf, true)));
    return fmaxf(x, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x121, 0xf, 0xf, true)));
}

// A value already divided by its block's scale, for the conversion: finite ones
// are at most 448 (or round to it), infinities become NaN (the format has none).
__device__ __forceinline__ float fp8_operand(float x) { return fabsf(x) < INFINITY ? x : NAN; }

// Two floats as codes in the low or the high half of `old`.
__device__ __forceinline__ uint32_t fp8_low(float a, float b) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(fp8_operand(a), fp8_operand(b), 0, false);
}
__device__ __forceinline__ uint32_t fp8_high(float a, float b, uint32_t old) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(fp8_operand(a), fp8_operand(b), (int)old, true);
}

// Eight values of a row, from column `col` on (a multiple of 8), as codes and,
// from the first of the 16 lanes that hold a block, its scale (and zeros past the
// last one). All lanes of a block call it, values past dim are zeros; `blocks` is
// fp8_blocks(dim).
// `amax` is the block's largest magnitude.
__device__ __forceinline__ void fp8_store8(const float (&v)[8], float amax, int64_t col, int64_t blocks, uint8_t* codes, uint8_t* scales) {
    const uint32_t byte = fp8_scale_byte(amax);
    const float inv = fp8_scale_inverse(byte);
    if (col < blocks * 128) {
        u32x2 w;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            w[i] = fp8_high(v[4 * i + 2] * inv, v[4 * i + 3] * inv, fp8_low(v[4 * i] * inv, v[4 * i + 1] * inv));
        *reinterpret_cast<u32x2*>(codes + col) = w;
    }
    if ((threadIdx.x & 15) == 0 && col < blocks * 128) {
        scales[col / 128] = (uint8_t)byte;
        if (col / 128 == blocks - 1)
            for (int64_t past = blocks; past < (blocks + 3) / 4 * 4; ++past) scales[past] = 0;
    }
}

__device__ __forceinline__ void fp8_store8(const float (&v)[8], int64_t col, int64_t blocks, uint8_t* codes, uint8_t* scales) {
    float amax = finite_magnitude(v[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) amax = fmaxf(amax, finite_magnitude(v[i]));
    fp8_store8(v, max_of_16(amax), col, blocks, codes, scales);
}

// Eight elements of a row from column `col` on, zeros from `dim` on, as loaded:
// what is made of them is made where they are used, so that several loads are on
// their way at once.
template <typename T>
struct Eight {
    u32x4 raw[sizeof(T) / 2];

    __device__ __forceinline__ void load(const T* p, int col, int dim) {
        if (col + 8 <= dim) {
            __builtin_memcpy(raw, p + col, sizeof raw);
            return;
        }
        typedef typename std::conditional<sizeof(T) == 2, uint16_t, uint32_t>::type U;
        const U* u = reinterpret_cast<const U*>(p);
        uint32_t t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = u[col + i < dim ? col + i : dim - 1];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i >= dim) t[i] = 0;
        if constexpr (sizeof(T) == 2) {
            raw[0] = u32x4{t[0] | t[1] << 16, t[2] | t[3] << 16, t[4] | t[5] << 16, t[6] | t[7] << 16};
        } else {
            raw[0] = u32x4{t[0], t[1], t[2], t[3]};
            raw[1] = u32x4{t[4], t[5], t[6], t[7]};
        }
    }
    // Element i; 16-bit ones are bfloat16 if `bf16`, else float16.
    __device__ __forceinline__ float get(int i, bool bf16 = std::is_same<T, __bf16>::value) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(raw[i / 4][i % 4]);
        const uint32_t pair = raw[0][i / 2];
        return bf16 ? bf16_of(pair, i % 2) : (float)__builtin_bit_cast(f16x2, pair)[i % 2];
    }
};

template <int N, typename T>
__device__ __forceinline__ void store_row(T* p, int64_t col, int64_t dim, const float (&v)[N]) {
    if (col + N <= dim) {
        T t[N];
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = (T)v[i];
        __builtin_memcpy(p + col, t, sizeof t);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (col + i < dim) p[col + i] = (T)v[i];
    }
}

}  // namespace tt
