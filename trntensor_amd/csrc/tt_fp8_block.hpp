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

// 2^(byte - 127); byte 255 is NaN.
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
    return __uint_as_float(byte == 0 ? 0x400000u : byte == 255 ? 0x7fc00000u : byte << 23);
}

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
// unit each, which costs nothing next to the products' sums (past a = -87 the
// exponential is infinite, and what would be below 10^-36 is 0); with a full division
// and exponential a round of tiles of 256 x 128 values took 14.2 us, with these 10.6
// (2048 x 16384 from one block of columns, four rounds: 56.6 and 42.6 us).
template <int ACTIVATION>
__device__ __forceinline__ float gate_value(float a, float b) {
    const float bend = ACTIVATION == 0 ? a : 1.5957691216f * (a + 0.044715f * a * a * a);
    return a * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504089f * bend)) * b;
}
__device__ __forceinline__ float gate_value(float a, float b, int activation) {
    return activation == 0 ? gate_value<0>(a, b) : gate_value<1>(a, b);
}

// A wavefront's part of a gated block's two products for one row and column, in 32
// bits: 16 columns of the operands a lane, from lane number `first` of `lanes` on. The
// sum of a wavefront's parts is in every lane.
template <bool E8, int UNROLL>
__device__ __forceinline__ void exact_parts(const Fp8Params& p, int row, int col, int first, int lanes, float (&sum)[2]) {
    const uint8_t* x = p.x + (int64_t)row * p.blocks * 128;
    const uint8_t* xs = p.xs + (int64_t)row * p.x_scales;
    const int64_t tile = (int64_t)(col / 16) * p.blocks * 2048 + col % 16 * 16;
    sum[0] = sum[1] = 0.f;
#pragma unroll UNROLL
    for (int piece = first; piece < p.blocks * 8; piece += lanes) {
        const int k = piece / 8, q = piece % 8;
        const u32x4 a = *reinterpret_cast<const u32x4*>(x + (int64_t)k * 128 + q * 16);
        const float scale = e8m0_value(xs[k]);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const u32x4 b = *reinterpret_cast<const u32x4*>(p.w[w] + tile + (int64_t)k * 2048 + q / 4 * 1024 + q % 4 * 256);
            const float ws = E8 ? e8m0_value(p.ws[w][(int64_t)(col / 128) * p.x_scales + k])
                                : reinterpret_cast<const float*>(p.ws[w])[(int64_t)(col / 128) * p.blocks + k];
            float part = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int ca = (int)a[i], cb = (int)b[i];
                part = __builtin_fmaf(__builtin_amdgcn_cvt_f32_fp8(ca, 0), __builtin_amdgcn_cvt_f32_fp8(cb, 0), part);
                part = __builtin_fmaf(__builtin_amdgcn_cvt_f32_fp8(ca, 1), __builtin_amdgcn_cvt_f32_fp8(cb, 1), part);
                part = __builtin_fmaf(__builtin_amdgcn_cvt_f32_fp8(ca, 2), __builtin_amdgcn_cvt_f32_fp8(cb, 2), part);
                part = __builtin_fmaf(__builtin_amdgcn_cvt_f32_fp8(ca, 3), __builtin_amdgcn_cvt_f32_fp8(cb, 3), part);
            }
            sum[w] += part * (scale * ws);
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        sum[0] += __shfl_xor(sum[0], off, kWave);
        sum[1] += __shfl_xor(sum[1], off, kWave);
    }
}

// The block's value there as a magnitude; 0 where it is not finite.
__device__ __forceinline__ float exact_gated(const float (&sum)[2], int activation) {
    return finite_magnitude(gate_value(sum[0], sum[1], activation));
}

// Values of the 8-bit matrix instructions are about 2^-16 of a sum off, which decides
// a block's scale where its largest value is next to 448 times a power of two:
// where it is within 2^-12 of that (one block in 1500), those of the block's values
// that come within 2^-11 of the largest are computed again in 32 bits, so that
// scales are those of 32-bit sums. A workgroup of tiles takes about 2 us longer
// for it (5 to 6 with a wavefront a value instead of all of them).
__device__ __forceinline__ bool near_border(float amax) {
    const int off = (int)(__float_as_uint(amax) & 0x7fffffu) - 0x600000;
    return off <= 3584 && off >= -3584 && amax >= 0x1p-100f;
}
constexpr float kCandidate = 1.f - 0x1p-11f;

// What a block's scale goes by where its largest value `amax` is near a border and
// `again` is that of the 32-bit sums: they say on which side of the border it lies,
// and no more. Where large terms cancel they can be anywhere, but the codes are
// made of the values that gave amax, which have to stay within the scale.
__device__ __forceinline__ float decided(float amax, float again) {
    return fminf(fmaxf(again, amax * kCandidate), amax * (1.f + 0x1p-11f));
}

// What a call's products are summed by and written as.
enum { kHalf, kExact, kRaw, kCodes };

// Workgroup tiles (tt_fp8_tiles.hip, tt_fp8_gated.hip): about how many us a call
// takes on the tile that is best for it, and that tile; the call on it.
double fp8_tiles_cost(const Fp8Params& p, bool exact, int* which);
int fp8_tiles(bool exact, bool e8, int which, const Fp8Params& p, hipStream_t st);
double fp8_gated_tiles_cost(const Fp8Params& p, int kind, int* which);
int fp8_gated_tiles(int kind, bool e8, int which, const Fp8Params& p, hipStream_t st);
// What kRaw wrote to y, into codes and scales.
int fp8_gated_round(bool e8, const Fp8Params& p, hipStream_t st);

}  // namespace tt
