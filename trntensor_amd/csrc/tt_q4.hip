// Products with 4-bit weights (tt_q4_matmul):
//   y[m][n] = sum_k x[m][k] s[k / g][n] (c[n][k] - z[k / g][n])
//
// Codes become 16-bit floats by two bit operations a pair: v = 1 + c / 16 has
// the code in the upper bits of its mantissa, in bfloat16 as in float16. With
// X the sum of x over a group, a group's share is then
//   16 s (sum x v - (1 + z / 16) X),
// where the matrix units form both sums (X as the product with ones) in 32
// bits; v lies in [1, 2), so that taking the offset off costs about two bits
// of the 24. An infinite x gives NaN or an infinity.
#include <type_traits>

#include "tt_serving.hpp"

namespace tt {

namespace {

struct Q4Params {
    int64_t ldx, ldy;
    const void *x, *scales, *zeros;
    const uint8_t* codes;
    void* y;
    int M, N, K, groups, chunks;  // chunks of 128 columns
    int group_shift, chunks_per_group;  // groups below 128 columns: log2(group / 32); else chunks a group
    int scale_bf16;                     // 16-bit scales: bfloat16, not float16
};

__device__ __forceinline__ f32x4 q4_mma(u32x4 a, u32x4 b, f32x4 c, __bf16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 q4_mma(u32x4 a, u32x4 b, f32x4 c, _Float16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// How activations enter the matrix units: 16-bit ones as they are, float32
// ones as three bfloat16 parts (24 bits).
template <typename T>
struct Act {
    typedef T half;
    static constexpr int parts = 1;
};
template <>
struct Act<float> {
    typedef __bf16 half;
    static constexpr int parts = 3;
};

// The eight codes of a packed word as v = 1 + c / 16, in their columns' order.
__device__ __forceinline__ u32x4 widen_codes(uint32_t w, __bf16) {
    u32x4 r;
    r[0] = ((w << 3) & 0x00780078u) | 0x3f803f80u;
    r[1] = ((w >> 1) & 0x00780078u) | 0x3f803f80u;
    r[2] = ((w >> 5) & 0x00780078u) | 0x3f803f80u;
    r[3] = ((w >> 9) & 0x00780078u) | 0x3f803f80u;
    return r;
}
__device__ __forceinline__ u32x4 widen_codes(uint32_t w, _Float16) {
    u32x4 r;
    r[0] = ((w << 6) & 0x03c003c0u) | 0x3c003c00u;
    r[1] = ((w << 2) & 0x03c003c0u) | 0x3c003c00u;
    r[2] = ((w >> 2) & 0x03c003c0u) | 0x3c003c00u;
    r[3] = ((w >> 6) & 0x03c003c0u) | 0x3c003c00u;
    return r;
}
__device__ __forceinline__ uint32_t one_pair(__bf16) { return 0x3f803f80u; }
__device__ __forceinline__ uint32_t one_pair(_Float16) { return 0x3c003c00u; }

// Scales or zero points of four neighbouring rows, as stored (SW bytes each).
template <int SW>
struct Four {
    uint32_t raw[SW];
    __device__ __forceinline__ f32x4 get(bool bf16) const {
        if constexpr (SW == 4)
            return f32x4{__uint_as_float(raw[0]), __uint_as_float(raw[1]), __uint_as_float(raw[2]), __uint_as_float(raw[3])};
        if (bf16)
            return f32x4{__uint_as_float(raw[0] << 16), __uint_as_float(raw[0] & 0xffff0000u), __uint_as_float(raw[1] << 16),
                         __uint_as_float(raw[1] & 0xffff0000u)};
        const f16x2 a = __builtin_bit_cast(f16x2, raw[0]), b = __builtin_bit_cast(f16x2, raw[1]);
        return f32x4{(float)a[0], (float)a[1], (float)b[0], (float)b[1]};
    }
};

constexpr int kWaves = 8;  // wavefronts a workgroup

// One stage of a wavefront's operands: a chunk of 128 columns of 16 R weight
// rows and 16 MT activation rows; GPC scales a chunk and row.
template <typename T, int SW, int R, int MT, int GPC>
struct Stage {
    u32x4 codes[R];
    Four<SW> scales[R][GPC], zeros[R][GPC];
    T x[MT][4][8];
};

// R blocks of 16 weight rows and MT of 16 activation rows a wavefront; the
// wavefronts of a workgroup take contiguous shares of the columns, which are
// summed at the end in their order. GPC: the pieces of a chunk of 128 columns
// that are scaled one by one, 1 for groups of at least a chunk, else 4.
template <typename T, int SW, int R, int MT, int GPC>
__global__ __launch_bounds__(64 * kWaves, 2) void q4_matmul_kernel(Q4Params p) {
    typedef typename Act<T>::half H;
    constexpr int NP = Act<T>::parts;
    constexpr int kSteps = 4 / GPC;  // MFMA steps of 32 columns a piece
    __shared__ float so[kWaves][MT * 16][R * 16 + 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int row_blocks = (p.N + 16 * R - 1) / (16 * R);
    const int m_blocks = (p.M + 16 * MT - 1) / (16 * MT);
    // Workgroup i runs on XCD i % 8: the blocks of activation rows that read
    // the same weights follow each other on one XCD, and share its L2.
    int rb, mb;
    const int tail = row_blocks % kNumXcd, whole = (row_blocks - tail) * m_blocks;
    if ((int)blockIdx.x < whole) {
        rb = blockIdx.x / (kNumXcd * m_blocks) * kNumXcd + blockIdx.x % kNumXcd;
        mb = blockIdx.x / kNumXcd % m_blocks;
    } else {
        rb = row_blocks - tail + (blockIdx.x - whole) % tail;
        mb = (blockIdx.x - whole) / tail;
    }
    const int n0 = rb * 16 * R, m0 = mb * 16 * MT;
    const int per = (p.chunks + kWaves - 1) / kWaves;
    const int first = wave * per, last = first + per < p.chunks ? first + per : p.chunks;

    // Rows past the end repeat the last ones: what they give is not stored.
    const int tiles = (p.N + 15) / 16;
    const uint8_t* code_row[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int t = rb * R + r;
        code_row[r] = p.codes + (int64_t)(t < tiles ? t : tiles - 1) * p.chunks * 1024 + lane * 16;
    }
    const T* x_row[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int m = m0 + mt * 16 + c;
        x_row[mt] = static_cast<const T*>(p.x) + (int64_t)(m < p.M ? m : p.M - 1) * p.ldx + g * 8;
    }
    // A last chunk that the columns do not fill, with zeros behind them.
    __shared__ __attribute__((aligned(16))) T filled[MT * 16][128 + 16 / sizeof(T)];
    const bool ragged = last == p.chunks && p.K % 128 != 0 && first < last;
    if (ragged) {
        const int k0 = (p.chunks - 1) * 128;
        for (int i = lane; i < MT * 16 * 128; i += 64) {
            const int m = m0 + i / 128, k = k0 + i % 128;
            filled[i / 128][i % 128] = k < p.K ? static_cast<const T*>(p.x)[(int64_t)(m < p.M ? m : p.M - 1) * p.ldx + k] : (T)0.f;
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    const bool bf16 = p.scale_bf16;
    const int scale_pitch = (p.N + 15) / 16 * 16;
    auto load_four = [&](const void* base, int group, int r) {
        Four<SW> f;
        group = group < p.groups ? group : p.groups - 1;
        const int n = n0 + r * 16 < scale_pitch ? n0 + r * 16 + g * 4 : 0;
        __builtin_memcpy(f.raw, static_cast<const uint8_t*>(base) + ((int64_t)group * scale_pitch + n) * SW, sizeof f.raw);
        return f;
    };
    typedef Stage<T, SW, R, MT, GPC> St;
    auto load = [&](St& st, int k) {
#pragma unroll
        for (int r = 0; r < R; ++r) st.codes[r] = *reinterpret_cast<const u32x4*>(code_row[r] + (int64_t)k * 1024);
        const bool edge = ragged && k == p.chunks - 1;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            if (edge) {
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    __builtin_memcpy(st.x[mt][s], __builtin_assume_aligned(&filled[mt * 16 + c][s * 32 + g * 8], 16),
                                     sizeof st.x[mt][s]);
            } else {
                const T* src = x_row[mt] + k * 128;
#pragma unroll
                for (int s = 0; s < 4; ++s) __builtin_memcpy(st.x[mt][s], src + s * 32, sizeof st.x[mt][s]);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int q = 0; q < GPC; ++q) {
                const int group = GPC > 1 ? (k * GPC + q) >> p.group_shift : k / p.chunks_per_group;
                st.scales[r][q] = load_four(p.scales, group, r);
                if (p.zeros) st.zeros[r][q] = load_four(p.zeros, group, r);
            }
    };
    f32x4 out[R][MT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) out[r][mt] = f32x4{0, 0, 0, 0};
    const uint32_t ones = one_pair(H());
    const u32x4 one = {ones, ones, ones, ones};
    auto fold = [&](const St& st) {
#pragma unroll
        for (int q = 0; q < GPC; ++q) {
            f32x4 sum[R][MT], total[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                total[mt] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int r = 0; r < R; ++r) sum[r][mt] = f32x4{0, 0, 0, 0};
            }
#pragma unroll
            for (int e = 0; e < kSteps; ++e) {
                const int s = q * kSteps + e;
                u32x4 b[MT][NP];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    if constexpr (NP == 1) {
                        b[mt][0] = __builtin_bit_cast(u32x4, st.x[mt][s]);
                    } else {
                        split8<NP>(st.x[mt][s], b[mt]);
                    }
#pragma unroll
                    for (int i = 0; i < NP; ++i) total[mt] = q4_mma(one, b[mt][i], total[mt], H());
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const u32x4 a = widen_codes(st.codes[r][s], H());
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int i = 0; i < NP; ++i) sum[r][mt] = q4_mma(a, b[mt][i], sum[r][mt], H());
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const f32x4 scale = st.scales[r][q].get(bf16) * 16.f;
                f32x4 off = {1.5f, 1.5f, 1.5f, 1.5f};
                if (p.zeros) off = st.zeros[r][q].get(bf16) * 0.0625f + 1.f;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) out[r][mt] += scale * (sum[r][mt] - off * total[mt]);
            }
        }
    };
    if (first < last) {
        St a, b;
        load(a, first);
        for (int k = first; k < last; k += 2) {
            if (k + 1 < last) load(b, k + 1);
            fold(a);
            if (k + 1 >= last) break;
            if (k + 2 < last) load(a, k + 2);
            fold(b);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) *reinterpret_cast<f32x4*>(&so[wave][mt * 16 + c][r * 16 + g * 4]) = out[r][mt];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * 16 * R * 4; i += 64 * kWaves) {
        const int m = i / (R * 4), n = i % (R * 4) * 4;
        if (m0 + m >= p.M || n0 + n >= p.N) continue;
        f32x4 v = *reinterpret_cast<const f32x4*>(&so[0][m][n]);
#pragma unroll
        for (int w = 1; w < kWaves; ++w) v += *reinterpret_cast<const f32x4*>(&so[w][m][n]);
        T* y = static_cast<T*>(p.y) + (int64_t)(m0 + m) * p.ldy + n0 + n;
        if (n0 + n + 4 <= p.N) {
            T t[4] = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
            __builtin_memcpy(y, t, sizeof t);
        } else {
            for (int j = 0; n0 + n + j < p.N; ++j) y[j] = (T)v[j];
        }
    }
}

template <typename T, int SW, int R, int MT, int GPC>
int q4_run(const Q4Params& p, hipStream_t st) {
    const int64_t grid = (int64_t)((p.N + 16 * R - 1) / (16 * R)) * ((p.M + 16 * MT - 1) / (16 * MT));
    if (grid > kMaxGrid / 4) return set_error(TT_UNSUPPORTED, "tt_q4_matmul: %lld workgroups", (long long)grid);
    q4_matmul_kernel<T, SW, R, MT, GPC><<<(uint32_t)grid, 64 * kWaves, 0, st>>>(p);
    return check_launch("tt_q4_matmul");
}

template <typename T, int SW, int GPC>
int q4_shape(const Q4Params& p, hipStream_t st) {
    // R weight tiles a wavefront read the same activations: fewer of their bytes
    // a byte of codes, but fewer wavefronts. us for R = 1 / 2 / 4 (bfloat16,
    // groups of 128): one row, 4096 x 4096 4.9 / 6.6 / 9.8, 8192 x 4096 7.4 /
    // 8.5 / 11.2, 16384 x 8192 20.4 / 18.1 / 20.1; 16 rows, 16384 x 8192 36.9 /
    // 24.5 / 22.7; 32 rows, 4096 x 4096 11.2 / 12.5 / 15.9, 16384 x 8192 69.9 /
    // 41.9 / 31.2. Four or sixteen wavefronts a workgroup, or two chunks a
    // stage, were slower at all of these or level.
    constexpr bool kWide = sizeof(T) == 4;  // three parts an activation: no room for two blocks of rows
    const int tiles = (p.N + 15) / 16;
    if (p.M <= 16 || kWide) {
        if (tiles <= 512) return q4_run<T, SW, 1, 1, GPC>(p, st);
        return q4_run<T, SW, 2, 1, GPC>(p, st);
    }
    if constexpr (!kWide) {
        if (tiles <= 256) return q4_run<T, SW, 1, 2, GPC>(p, st);
        return q4_run<T, SW, GPC == 1 ? 4 : 2, 2, GPC>(p, st);
    }
    return TT_OK;
}

template <typename T>
int q4_typed(int64_t scale_dtype, const Q4Params& p, bool small_groups, hipStream_t st) {
    if (scale_dtype == TT_F32) return small_groups ? q4_shape<T, 4, 4>(p, st) : q4_shape<T, 4, 1>(p, st);
    return small_groups ? q4_shape<T, 2, 4>(p, st) : q4_shape<T, 2, 1>(p, st);
}

// One thread a lane's 16 bytes of a tile.
__global__ __launch_bounds__(256) void q4_pack_kernel(int N, int K, int chunks, const uint8_t* codes, int64_t pitch,
                                                      u32x4* out, int64_t count) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= count) return;
    const int lane = i & 63;
    const int64_t tile = i >> 6;
    const int chunk = (int)(tile % chunks);
    const int64_t n = tile / chunks * 16 + (lane & 15);
    const int bytes = (K + 1) / 2;
    u32x4 w;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int at = chunk * 64 + s * 16 + (lane >> 4) * 4;
        uint32_t x = 0;
        if (n < N && at + 4 <= bytes) {
            __builtin_memcpy(&x, codes + n * pitch + at, 4);
        } else if (n < N) {
            for (int j = 0; at + j < bytes; ++j) x |= (uint32_t)codes[n * pitch + at + j] << 8 * j;
        }
        uint32_t even = x & 0x0f0f0f0fu, odd = x >> 4 & 0x0f0f0f0fu;
        even = (even | even >> 4) & 0x00ff00ffu;
        odd = (odd | odd >> 4) & 0x00ff00ffu;
        w[s] = ((even | even >> 8) & 0xffffu) | (odd | odd >> 8) << 16;
    }
    out[i] = w;
}

int check_q4_size(const char* who, int64_t N, int64_t K) {
    constexpr int64_t kMost = int64_t(1) << 30;
    if (N < 0 || K < 1) return set_error(TT_INVALID, "%s: %lld rows of %lld columns", who, (long long)N, (long long)K);
    if (N > kMost || K > kMost) return set_error(TT_UNSUPPORTED, "%s: extents beyond 2^30", who);
    return TT_OK;
}

}  // namespace
}  // namespace tt

extern "C" size_t tt_q4_packed_bytes(int64_t N, int64_t K) {
    if (N < 1 || K < 1) return 0;
    return (size_t)((N + 15) / 16) * (size_t)((K + 127) / 128) * 1024;
}

extern "C" int tt_q4_pack(int64_t N, int64_t K, const void* codes, int64_t pitch, void* packed, void* stream) {
    using namespace tt;
    if (int rc = check_q4_size("tt_q4_pack", N, K)) return rc;
    if (N == 0) return TT_OK;
    if (!codes || !packed) return set_error(TT_INVALID, "tt_q4_pack: NULL pointer");
    if (pitch < (K + 1) / 2 || (uintptr_t)packed % 16)
        return set_error(TT_INVALID, "tt_q4_pack: pitch %lld, or alignment", (long long)pitch);
    const int64_t count = (int64_t)(tt_q4_packed_bytes(N, K) / 16), blocks = (count + 255) / 256;
    if (blocks > kMaxGrid) return set_error(TT_UNSUPPORTED, "tt_q4_pack: %lld by %lld codes", (long long)N, (long long)K);
    q4_pack_kernel<<<(uint32_t)blocks, 256, 0, static_cast<hipStream_t>(stream)>>>(
        (int)N, (int)K, (int)((K + 127) / 128), static_cast<const uint8_t*>(codes), pitch, static_cast<u32x4*>(packed), count);
    return check_launch("tt_q4_pack");
}

extern "C" int tt_q4_matmul(const tt_q4_args* a, void* stream) {
    using namespace tt;
    if (!a) return set_error(TT_INVALID, "tt_q4_matmul: NULL arguments");
    if (!serving_dtype(a->dtype) || !serving_dtype(a->scale_dtype))
        return set_error(TT_UNSUPPORTED, "tt_q4_matmul: dtypes %lld, %lld (TT_F32, TT_BF16, TT_F16)",
                         (long long)a->dtype, (long long)a->scale_dtype);
    if (int rc = check_q4_size("tt_q4_matmul", a->N, a->K)) return rc;
    if (a->M < 0) return set_error(TT_INVALID, "tt_q4_matmul: %lld rows", (long long)a->M);
    if (a->M > int64_t(1) << 30) return set_error(TT_UNSUPPORTED, "tt_q4_matmul: extents beyond 2^30");
    if (a->group != 32 && a->group != 64 && (a->group < 128 || a->group % 128))
        return set_error(TT_INVALID, "tt_q4_matmul: group of %lld (32, 64 or a multiple of 128)", (long long)a->group);
    if (a->M == 0 || a->N == 0) return TT_OK;
    if (!a->y || !a->x || !a->codes || !a->scales) return set_error(TT_INVALID, "tt_q4_matmul: NULL pointer");
    if (a->ldx < a->K || a->ldy < a->N) return set_error(TT_INVALID, "tt_q4_matmul: leading dimension below the width");
    if (((uintptr_t)a->codes | (uintptr_t)a->scales | (uintptr_t)a->zeros) % 16)
        return set_error(TT_INVALID, "tt_q4_matmul: weights are not 16-byte aligned");
    Q4Params p;
    p.ldx = a->ldx;
    p.ldy = a->ldy;
    p.x = a->x;
    p.scales = a->scales;
    p.zeros = a->zeros;
    p.codes = static_cast<const uint8_t*>(a->codes);
    p.y = a->y;
    p.M = (int)a->M;
    p.N = (int)a->N;
    p.K = (int)a->K;
    const int64_t group = a->group < a->K ? a->group : (a->K + 127) / 128 * 128;  // a single one: whole chunks
    p.groups = (int)((a->K + a->group - 1) / a->group);
    p.chunks = (int)((a->K + 127) / 128);
    p.chunks_per_group = group >= 128 ? (int)(group / 128) : 1;
    p.group_shift = group == 64 ? 1 : 0;
    p.scale_bf16 = a->scale_dtype == TT_BF16;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->dtype == TT_F32) return q4_typed<float>(a->scale_dtype, p, group < 128, st);
    if (a->dtype == TT_BF16) return q4_typed<__bf16>(a->scale_dtype, p, group < 128, st);
    return q4_typed<_Float16>(a->scale_dtype, p, group < 128, st);
}
