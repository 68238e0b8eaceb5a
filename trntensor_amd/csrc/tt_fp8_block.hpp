// Operands and products of the 8-bit chain's matrix kernels (tt_fp8.hip,
// tt_fp8_tiles.hip).
#pragma once

#include "tt_fp8.hpp"

namespace tt {

typedef int i32x8 __attribute__((ext_vector_type(8)));

struct Fp8Params {
    const uint8_t *x, *xs;       // rows and their scales
    const uint8_t *w[2], *ws[2]; // weights (gate and up)
    void* y;
    uint8_t *codes, *scales;
    int M, N, K, blocks, x_scales;  // blocks of 128 columns; scale bytes of a row
    int activation;
    int bf16;  // 16-bit results are bfloat16
};

constexpr uint32_t kOne = 127;  // e8m0 of 1.0

// out += scales * A B^T for 16 rows of either and a block of 128 columns, A being
// weights. The 8-bit matrix instructions take eight products at a time, align
// them to the largest and drop what lies 2^-13 below its power of two (measured;
// sums of eights are added in 24 bits). For results of 16 and 8 bits that is
// nothing: 2^-16 of a sum of 128 terms of normal distribution. Exact ones
// (float32 results) have the codes widened to bfloat16, whose products the
// matrix units add in 32 bits at half the rate.
template <bool EXACT, bool E8>
struct Block {
    u32x4 v[2];

    __device__ __forceinline__ void load(const uint8_t* first, const uint8_t* second) {
        v[0] = *reinterpret_cast<const u32x4*>(first);
        v[1] = *reinterpret_cast<const u32x4*>(second);
    }
    __device__ __forceinline__ i32x8 operand() const {
        return i32x8{(int)v[0][0], (int)v[0][1], (int)v[0][2], (int)v[0][3], (int)v[1][0], (int)v[1][1], (int)v[1][2], (int)v[1][3]};
    }
    // Eight codes as bfloat16.
    __device__ __forceinline__ bf16x8 wide(int i) const {
        u32x4 r;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t c = v[i / 2][i % 2 * 2 + j];
            r[2 * j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.f, false));
            r[2 * j + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.f, true));
        }
        return __builtin_bit_cast(bf16x8, r);
    }
};

__device__ __forceinline__ float e8m0_value(uint32_t byte) { return byte ? __uint_as_float(byte << 23) : 0x1p-127f; }

// The sum of a block of 128 columns with the scales of x's rows alone.
template <bool EXACT, bool E8>
__device__ __forceinline__ f32x4 block_sum(const Block<EXACT, E8>& a, const Block<EXACT, E8>& b, uint32_t sb) {
    const f32x4 zero = {0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.operand(), b.operand(), zero, 0, 0, 0, kOne, 0, (int)sb);
}

// `sa`: the weights' scale, a byte or a float's bits; `sb`: the byte of this lane's row of x.
template <bool EXACT, bool E8>
__device__ __forceinline__ void mma_block(const Block<EXACT, E8>& a, const Block<EXACT, E8>& b, f32x4& out, uint32_t sa, uint32_t sb) {
    if constexpr (EXACT) {
        f32x4 sum = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.wide(i), b.wide(i), sum, 0, 0, 0);
        out += (E8 ? e8m0_value(sa) : __uint_as_float(sa)) * e8m0_value(sb) * sum;
    } else if constexpr (E8) {
        out = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.operand(), b.operand(), out, 0, 0, 0, (int)sa, 0, (int)sb);
    } else {
        out += __uint_as_float(sa) * block_sum(a, b, sb);
    }
}

// The scale of a block of weights, as mma_block takes it: a scalar load, so
// that no wait for it is one for the vector loads on their way.
template <bool E8>
__device__ __forceinline__ uint32_t weight_scale(const Fp8Params& p, int r, int tile, int k) {
    typedef const __attribute__((address_space(4))) uint32_t constant_word;
    const int64_t at = E8 ? (int64_t)(tile / 8) * (p.x_scales / 4) + k / 4 : (int64_t)(tile / 8) * p.blocks + k;
    const uint32_t word = ((constant_word*)(uintptr_t)p.ws[r])[at];
    return E8 ? word >> (k & 3) * 8 & 255 : word;
}

// act(a) b: both activations are a / (1 + exp(-bend)), since (1 + tanh(z)) / 2 is 1 /
// (1 + exp(-2 z)). The hardware's exponential (of base 2) and reciprocal err by a
// unit each, which costs nothing next to the products' sums; with a full division
// and exponential a tile of 256 x 128 values took 14 us for @ beside its products.
template <int ACTIVATION>
__device__ __forceinline__ float gate_value(float a, float b) {
    const float bend = ACTIVATION == 0 ? a : 1.5957691216f * (a + 0.044715f * a * a * a);
    return a * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504089f * bend)) * b;
}
__device__ __forceinline__ float gate_value(float a, float b, int activation) {
    return activation == 0 ? gate_value<0>(a, b) : gate_value<1>(a, b);
}

// What a call's products are summed by and written as.
enum { kHalf, kExact, kRaw, kCodes };

// Workgroup tiles (tt_fp8_tiles.hip, tt_fp8_gated.hip): about how many us a call
// takes on the tile that is best for it, and that tile; the call on it.
double fp8_tiles_cost(const Fp8Params& p, bool exact, int* which);
int fp8_tiles(bool exact, bool e8, int which, const Fp8Params& p, hipStream_t st);
double fp8_gated_tiles_cost(const Fp8Params& p, int kind, int* which);
int fp8_gated_tiles(int kind, bool e8, int which, const Fp8Params& p, hipStream_t st);

}  // namespace tt
