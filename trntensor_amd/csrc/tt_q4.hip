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

constexpr int KW = 8;  // wavefronts a workgroup

struct Q4Params {
    int64_t ldx, code_pitch, ldy;
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

// Eight codes of one word (code i in bits 4 i ..) as v = 1 + c / 16, in the
// order 0 4 1 5 2 6 3 7.
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

// Eight 16-bit values in the codes' order.
__device__ __forceinline__ u32x4 code_order(u32x4 x) {
    u32x4 r;
    r[0] = __builtin_amdgcn_perm(x[2], x[0], 0x05040100u);
    r[1] = __builtin_amdgcn_perm(x[2], x[0], 0x07060302u);
    r[2] = __builtin_amdgcn_perm(x[3], x[1], 0x05040100u);
    r[3] = __builtin_amdgcn_perm(x[3], x[1], 0x07060302u);
    return r;
}

// Exchanges word i of lane group j with word j of lane group i (groups of 16
// lanes): a lane that read 16 bytes of a row then holds, word by word, its part
// of four runs of 32 columns instead of one run of its own.
__device__ __forceinline__ u32x4 swap_words(u32x4 x) {
    auto a = __builtin_amdgcn_permlane32_swap(x[0], x[2], false, false);
    auto b = __builtin_amdgcn_permlane32_swap(x[1], x[3], false, false);
    auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return u32x4{c[0], c[1], d[0], d[1]};
}

// Scales or zero points of four neighbouring rows, as stored (SW bytes each).
template <int SW>
struct Four {
    uint32_t raw[SW];
    __device__ __forceinline__ float get(int i, bool bf16) const {
        if constexpr (SW == 4) return __uint_as_float(raw[i]);
        const uint32_t h = i & 1 ? raw[i / 2] >> 16 : raw[i / 2] & 0xffffu;
        return bf16 ? __uint_as_float(h << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
    }
};

// One stage of a wavefront's operands: U chunks of 128 columns of 16 R weight
// rows and 16 MT activation rows; GPC scales a chunk and row.
template <typename T, int SW, int U, int R, int MT, int GPC>
struct Stage {
    u32x4 codes[U][R];
    Four<SW> scales[U][R][GPC], zeros[U][R][GPC];
    T x[U][MT][4][8];
};

// R blocks of 16 weight rows and MT of 16 activation rows a wavefront; the KW
// wavefronts of a workgroup take contiguous shares of the columns, which are
// summed at the end in their order. GPC: the pieces of a chunk of 128 columns
// that are scaled one by one, 1 for groups of at least a chunk, else 4.
template <typename T, int SW, int U, int R, int MT, int GPC>
__global__ __launch_bounds__(64 * KW, 2) void q4_matmul_kernel(Q4Params p) {
    typedef typename Act<T>::half H;
    constexpr int NP = Act<T>::parts;
    constexpr int kSteps = 4 / GPC;  // MFMA steps of 32 columns a piece
    __shared__ float so[KW][MT * 16][R * 16 + 4];
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
    const int per = (p.chunks + KW - 1) / KW;
    const int first = wave * per, last = first + per < p.chunks ? first + per : p.chunks;

    // Rows past the end repeat the last one: what they give is not stored.
    const uint8_t* code_row[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int n = n0 + r * 16 + c;
        code_row[r] = p.codes + (int64_t)(n < p.N ? n : p.N - 1) * p.code_pitch + g * 16;
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
    typedef Stage<T, SW, U, R, MT, GPC> St;
    auto load = [&](St& st, int chunk) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = chunk + u < last ? chunk + u : last - 1;
#pragma unroll
            for (int r = 0; r < R; ++r) st.codes[u][r] = *reinterpret_cast<const u32x4*>(code_row[r] + (int64_t)k * 64);
            const bool edge = ragged && k == p.chunks - 1;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                if (edge) {
#pragma unroll
                    for (int s = 0; s < 4; ++s)
                        __builtin_memcpy(st.x[u][mt][s], __builtin_assume_aligned(&filled[mt * 16 + c][s * 32 + g * 8], 16),
                                         sizeof st.x[u][mt][s]);
                } else {
                    const T* src = x_row[mt] + k * 128;
#pragma unroll
                    for (int s = 0; s < 4; ++s) __builtin_memcpy(st.x[u][mt][s], src + s * 32, sizeof st.x[u][mt][s]);
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int q = 0; q < GPC; ++q) {
                    const int group = GPC > 1 ? (k * GPC + q) >> p.group_shift : k / p.chunks_per_group;
                    st.scales[u][r][q] = load_four(p.scales, group, r);
                    if (p.zeros) st.zeros[u][r][q] = load_four(p.zeros, group, r);
                }
        }
    };
    f32x4 out[R][MT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) out[r][mt] = f32x4{0, 0, 0, 0};
    const uint32_t ones = one_pair(H());
    const u32x4 one = {ones, ones, ones, ones};
    auto fold = [&](const St& st, int chunk) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (chunk + u >= last) break;
            u32x4 w[R];
#pragma unroll
            for (int r = 0; r < R; ++r) w[r] = swap_words(st.codes[u][r]);
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
                            b[mt][0] = code_order(__builtin_bit_cast(u32x4, st.x[u][mt][s]));
                        } else {
                            u32x4 part[NP];
                            split8<NP>(st.x[u][mt][s], part);
#pragma unroll
                            for (int i = 0; i < NP; ++i) b[mt][i] = code_order(part[i]);
                        }
#pragma unroll
                        for (int i = 0; i < NP; ++i) total[mt] = q4_mma(one, b[mt][i], total[mt], H());
                    }
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const u32x4 a = widen_codes(w[r][s], H());
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                            for (int i = 0; i < NP; ++i) sum[r][mt] = q4_mma(a, b[mt][i], sum[r][mt], H());
                    }
                }
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float sc = 16.f * st.scales[u][r][q].get(i, bf16);
                        const float off = p.zeros ? 1.f + 0.0625f * st.zeros[u][r][q].get(i, bf16) : 1.5f;
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) out[r][mt][i] += sc * (sum[r][mt][i] - off * total[mt][i]);
                    }
            }
        }
    };
    if (first < last) {
        St a, b;
        load(a, first);
        for (int k = first; k < last; k += 2 * U) {
            if (k + U < last) load(b, k + U);
            fold(a, k);
            if (k + U >= last) break;
            if (k + 2 * U < last) load(a, k + 2 * U);
            fold(b, k + U);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) *reinterpret_cast<f32x4*>(&so[wave][mt * 16 + c][r * 16 + g * 4]) = out[r][mt];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * 16 * R * 4; i += 64 * KW) {
        const int m = i / (R * 4), n = i % (R * 4) * 4;
        if (m0 + m >= p.M || n0 + n >= p.N) continue;
        f32x4 v = *reinterpret_cast<const f32x4*>(&so[0][m][n]);
#pragma unroll
        for (int w = 1; w < KW; ++w) v += *reinterpret_cast<const f32x4*>(&so[w][m][n]);
        T* y = static_cast<T*>(p.y) + (int64_t)(m0 + m) * p.ldy + n0 + n;
        if (n0 + n + 4 <= p.N) {
            T t[4] = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
            __builtin_memcpy(y, t, sizeof t);
        } else {
            for (int j = 0; n0 + n + j < p.N; ++j) y[j] = (T)v[j];
        }
    }
}

template <typename T, int SW, int U, int R, int MT, int GPC>
int q4_run(const Q4Params& p, hipStream_t st) {
    const int64_t grid = (int64_t)((p.N + 16 * R - 1) / (16 * R)) * ((p.M + 16 * MT - 1) / (16 * MT));
    if (grid > kMaxGrid / 2) return set_error(TT_UNSUPPORTED, "tt_q4_matmul: %lld workgroups", (long long)grid);
    q4_matmul_kernel<T, SW, U, R, MT, GPC><<<(uint32_t)grid, 64 * KW, 0, st>>>(p);
    return check_launch("tt_q4_matmul");
}

template <typename T, int SW, int GPC>
int q4_shape(const Q4Params& p, hipStream_t st) {
    constexpr bool kWide = sizeof(T) == 4;  // three parts an activation: no room for two blocks of rows
    if (p.N <= 8192 && (p.M <= 16 || kWide)) return q4_run<T, SW, kWide ? 1 : 2, 1, 1, GPC>(p, st);
    if (p.M <= 16 || kWide) return q4_run<T, SW, 1, 2, 1, GPC>(p, st);
    if constexpr (!kWide) return q4_run<T, SW, 1, 2, 2, GPC>(p, st);
    return TT_OK;
}

template <typename T>
int q4_typed(int64_t scale_dtype, const Q4Params& p, bool small_groups, hipStream_t st) {
    if (scale_dtype == TT_F32) return small_groups ? q4_shape<T, 4, 4>(p, st) : q4_shape<T, 4, 1>(p, st);
    return small_groups ? q4_shape<T, 2, 4>(p, st) : q4_shape<T, 2, 1>(p, st);
}

}  // namespace
}  // namespace tt

extern "C" size_t tt_q4_matmul_workspace_bytes(int dtype, int64_t M, int64_t N, int64_t K) {
    (void)dtype, (void)M, (void)N, (void)K;
    return 0;
}

extern "C" int tt_q4_matmul(const tt_q4_args* a, void* stream) {
    using namespace tt;
    if (!a) return set_error(TT_INVALID, "tt_q4_matmul: NULL arguments");
    if (!serving_dtype(a->dtype) || !serving_dtype(a->scale_dtype))
        return set_error(TT_UNSUPPORTED, "tt_q4_matmul: dtypes %lld, %lld (TT_F32, TT_BF16, TT_F16)",
                         (long long)a->dtype, (long long)a->scale_dtype);
    if (a->M < 0 || a->N < 0 || a->K < 1)
        return set_error(TT_INVALID, "tt_q4_matmul: extents %lld, %lld, %lld", (long long)a->M, (long long)a->N,
                         (long long)a->K);
    if (a->group != 32 && a->group != 64 && (a->group < 128 || a->group % 128))
        return set_error(TT_INVALID, "tt_q4_matmul: group of %lld (32, 64 or a multiple of 128)", (long long)a->group);
    if (a->M == 0 || a->N == 0) return TT_OK;
    if (!a->y || !a->x || !a->codes || !a->scales) return set_error(TT_INVALID, "tt_q4_matmul: NULL pointer");
    if (a->ldx < a->K || a->ldy < a->N) return set_error(TT_INVALID, "tt_q4_matmul: leading dimension below the width");
    if (a->code_pitch % 64 || a->code_pitch < (a->K + 1) / 2 || (uintptr_t)a->codes % 16)
        return set_error(TT_INVALID, "tt_q4_matmul: code pitch %lld or alignment", (long long)a->code_pitch);
    constexpr int64_t kMost = int64_t(1) << 30;
    if (a->M > kMost || a->N > kMost || a->K > kMost)
        return set_error(TT_UNSUPPORTED, "tt_q4_matmul: extents beyond 2^30");
    Q4Params p;
    p.ldx = a->ldx;
    p.code_pitch = a->code_pitch;
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
