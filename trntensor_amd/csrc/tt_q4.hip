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
    uint32_t zero_mask;                 // all ones where there are zero points, else 0 (and `zeros` is `scales`)
    uint32_t scale_bf16;                // 16-bit scales: all ones for bfloat16, 0 for float16
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
    uint32_t raw __attribute__((ext_vector_type(SW)));
    // 16-bit ones are bfloat16 where the bits of `bf16` are set, else float16
    // (not a condition: the compiler would gather all conversions under one
    // branch, and the floats with them).
    __device__ __forceinline__ f32x4 get(uint32_t bf16) const {
        if constexpr (SW == 4)
            return f32x4{__uint_as_float(raw[0]), __uint_as_float(raw[1]), __uint_as_float(raw[2]), __uint_as_float(raw[3])};
        f32x4 v;
        if constexpr (SW == 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t pair = raw[i / 2];
                const float half = (float)__builtin_bit_cast(f16x2, pair)[i & 1];
                v[i] = __uint_as_float((__float_as_uint(bf16_of(pair, i & 1)) & bf16) | (__float_as_uint(half) & ~bf16));
            }
        }
        return v;
    }
};

constexpr int kWaves = 8;  // wavefronts a workgroup

// What a wavefront holds of a chunk of 128 columns of its 16 R weight rows: codes
// and, for GPC pieces of the chunk, scales and zero points (or scales again).
template <int SW, int R, int GPC>
struct Chunk {
    u32x4 codes[R];
    Four<SW> scales[R][GPC], zeros[R][GPC];
};

// R blocks of 16 weight rows and MT of 16 activation rows a wavefront; the
// wavefronts of a workgroup take contiguous shares of the columns, which are
// summed at the end in their order: a row's codes are read once, as 1 KiB a
// load, by as many wavefronts as there are CUs to hold them. A few rows are
// bound by the codes' bytes (1 row on 16384 x 8192: 16.9 us where they take 14;
// on 4096 x 4096, 4.6 us, by the launch and three waits on memory one after the
// other; between them by whole rounds of workgroups on the CUs: 12288, 14336 and
// 16384 x 4096 take 12.1, 12.4 and 12.8 us), more by the vector units: 32 rows on 16384 x 8192 take 27 us, in which
// a wavefront issues 448 vector instructions a chunk (codes widened, scales and
// zero points made floats of either type and applied) beside 40 products. They
// issue 56% of a SIMD's time, and keep the matrix unit busy 18%; the 212 MB
// that leave L2 are 8 TB/s. Groups of 32 and 64 scale four pieces a chunk (57
// us), and every 32 rows widen all codes again: 2048 rows on 4096 x 4096 take 206
// us, 0.33 PFLOP/s (groups of 64: 475 us). GPC: the pieces of a chunk of 128
// columns that are scaled one by one, 1 for groups of at least a chunk, else 4.
template <typename T, int SW, int R, int MT, int GPC>
__global__ __launch_bounds__(64 * kWaves, 2) void q4_matmul_kernel(Q4Params p) {
    typedef typename Act<T>::half H;
    constexpr int NP = Act<T>::parts;
    constexpr int kSteps = 4 / GPC;  // MFMA steps of 32 columns a piece
    __shared__ float so[kWaves][MT * 16][R * 16 + 4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const int row_blocks = (p.N + 16 * R - 1) / (16 * R);
    const int m_blocks = (p.M + 16 * MT - 1) / (16 * MT);
    // Workgroup i runs on XCD i % 8: the blocks of activation rows that read
    // the same weights follow each other on one XCD, and share its L2.
    int rb, mb;
    const int tail = row_blocks % kNumXcd, even = (row_blocks - tail) * m_blocks;
    if ((int)blockIdx.x < even) {
        rb = blockIdx.x / (kNumXcd * m_blocks) * kNumXcd + blockIdx.x % kNumXcd;
        mb = blockIdx.x / kNumXcd % m_blocks;
    } else {
        rb = row_blocks - tail + (blockIdx.x - even) % tail;
        mb = (blockIdx.x - even) / tail;
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
        code_row[r] = p.codes + (int64_t)(t < tiles ? t : tiles - 1) * p.chunks * 1024;
    }
    const T* x_row[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int m = m0 + mt * 16 + c;
        x_row[mt] = static_cast<const T*>(p.x) + (int64_t)(m < p.M ? m : p.M - 1) * p.ldx + g * 8;
    }
    // A last chunk that the columns do not fill, with zeros behind them.
    __shared__ __attribute__((aligned(16))) T filled[MT * 16][128 + 16 / sizeof(T)];
    const bool uneven = p.K % 128 != 0, ragged = uneven && last == p.chunks && first < last;
    const int whole = ragged ? last - 1 : last;
    if (uneven) {
        constexpr int kEach = MT * 16 * 128 / (64 * kWaves);
        const int k = (p.chunks - 1) * 128 + threadIdx.x % 128;
        T v[kEach];
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
            const int m = m0 + u * (64 * kWaves / 128) + threadIdx.x / 128;
            v[u] = static_cast<const T*>(p.x)[(int64_t)(m < p.M ? m : p.M - 1) * p.ldx + (k < p.K ? k : p.K - 1)];
        }
#pragma unroll
        for (int u = 0; u < kEach; ++u)
            filled[u * (64 * kWaves / 128) + threadIdx.x / 128][threadIdx.x % 128] = k < p.K ? v[u] : (T)0.f;
    }
    const uint32_t bf16 = p.scale_bf16, eight = __float_as_uint(8.f);
    const int scale_pitch = (p.N + 15) / 16 * 16;
    auto load_four = [&](const void* base, int group, int r) {
        Four<SW> f;
        group = group < p.groups ? group : p.groups - 1;
        const int n = n0 + r * 16 < scale_pitch ? n0 + r * 16 : 0;
        f.raw = *reinterpret_cast<const decltype(f.raw)*>(static_cast<const uint8_t*>(base) +
                                                          ((int64_t)group * scale_pitch + n) * SW + (uint32_t)(g * 4 * SW));
        return f;
    };
    auto load = [&](Chunk<SW, R, GPC>& w, int k) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < R; ++r) w.codes[r] = *reinterpret_cast<const u32x4*>(code_row[r] + (int64_t)k * 1024 + (uint32_t)(lane * 16));
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int q = 0; q < GPC; ++q) {
                const int group = GPC > 1 ? (k * GPC + q) >> p.group_shift : k / p.chunks_per_group;
                w.scales[r][q] = load_four(p.scales, group, r);
                w.zeros[r][q] = load_four(p.zeros, group, r);
            }
        __builtin_amdgcn_sched_barrier(0);
    };
    T x[MT][4][8];
    auto load_x = [&](int s, int k) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) __builtin_memcpy(x[mt][s], x_row[mt] + k * 128 + s * 32, sizeof x[mt][s]);
    };
    f32x4 out[R][MT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) out[r][mt] = f32x4{0, 0, 0, 0};
    const uint32_t ones = one_pair(H());
    const u32x4 one = {ones, ones, ones, ones};
    // Folds a chunk; the activations of chunk `next` take the place of each step's.
    auto fold = [&](const Chunk<SW, R, GPC>& w, int next, auto reload) {
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
                        b[mt][0] = __builtin_bit_cast(u32x4, x[mt][s]);
                    } else {
                        split8<NP>(x[mt][s], b[mt]);
                    }
#pragma unroll
                    for (int i = 0; i < NP; ++i) total[mt] = q4_mma(one, b[mt][i], total[mt], H());
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const u32x4 a = widen_codes(w.codes[r][s], H());
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int i = 0; i < NP; ++i) sum[r][mt] = q4_mma(a, b[mt][i], sum[r][mt], H());
                }
                if constexpr (reload.value) load_x(s, next);
            }
            __builtin_amdgcn_sched_barrier(0);  // scales become floats here, not earlier
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const f32x4 scale = w.scales[r][q].get(bf16) * 16.f;
                f32x4 off = w.zeros[r][q].get(bf16);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    off[i] = __builtin_fmaf(__uint_as_float((__float_as_uint(off[i]) & p.zero_mask) | (eight & ~p.zero_mask)),
                                            0.0625f, 1.f);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) out[r][mt] += scale * (sum[r][mt] - off * total[mt]);
            }
        }
    };
    // A chunk is folded with the next one in flight, loaded into the other of a
    // and b; the last is in a, so that an odd number of steps begins with b. No
    // load hangs on a condition of its own: a wait for one chunk would become one
    // for all. (Loading the last chunk twice instead costs a wait at the end.)
    Chunk<SW, R, GPC> a, b;
    const int final = whole - 1;
    if (first <= final) {
        int second = (final - first) & 1;
        asm volatile("" : "+s"(second));
        if (second)
            load(b, first);
        else
            load(a, first);
#pragma unroll
        for (int s = 0; s < 4; ++s) load_x(s, first);
        for (int k = first; k < final;) {
            if (!second) {
                load(b, ++k);
                fold(a, k, std::true_type());
            }
            second = 0;
            asm volatile("" : "+s"(second));
            load(a, ++k);
            fold(b, k, std::true_type());
        }
    }
    if (uneven) __syncthreads();
    // The last whole chunk, and then the one that the columns do not fill.
    for (int left = (first < whole) + ragged; left > 0; --left) {
        if (ragged && left == 1) {
            load(a, p.chunks - 1);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    __builtin_memcpy(x[mt][s], __builtin_assume_aligned(&filled[mt * 16 + c][s * 32 + g * 8], 16),
                                     sizeof x[mt][s]);
        }
        fold(a, 0, std::false_type());
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
    // R weight tiles a wavefront share its activations: less of them to read and
    // to split, but fewer workgroups. `work` counts those of R = 1, of which two
    // fit a compute unit, and one of the others. us for R = 1 / 2 / 4:
    //   bfloat16, groups of 128        work 256          512              1024
    //     1 row     (K 4096, 4096, 8192)  5.2 / 6.5 / 9.8   7.4 / 8.1 / 10.8   20.3 / 16.9 / 20.4
    //     16 rows                         7.0 / 7.8 / 10.8  11.2 / 9.2 / 11.4  35.8 / 22.6 / 21.4
    //     32 rows                         10.4 / 11.2 / 13.9  18.0 / 12.4 / 14.8  63.1 / 37.6 / 27.0
    //   16-bit, groups of 64 and 32, zero points                                       1792 (K 4096)
    //     1 row                           8.8 / 13.8        13.2 / 14.8        40.0 / 43.1        36.3 / 49.0
    //     16 rows                         9.3 / 14.3        15.4 / 15.0        49.5 / 44.4        43.4 / 51.4
    //     32 rows                         12.7 / 17.1       23.2 / 17.8        82.2 / 56.9        76.8 / 64.1
    //     (up to 16 rows stay at R = 1: 2 gains 10% at 1024 and loses 18% at 1792, which no bound on work tells apart)
    //   float32 (three parts an activation: no room for two blocks of rows), groups of 32
    //     1 row                           9.9 / 13.2        18.5 / 15.9        59.2 / 48.1
    // Four or sixteen wavefronts a workgroup were slower or level.
    const int64_t tiles = (p.N + 15) / 16;
    if constexpr (sizeof(T) == 4) {
        if (tiles * ((p.M + 15) / 16) <= 256) return q4_run<T, SW, 1, 1, GPC>(p, st);
        return q4_run<T, SW, 2, 1, GPC>(p, st);
    } else if constexpr (GPC > 1) {
        if (p.M <= 16) return q4_run<T, SW, 1, 1, GPC>(p, st);
        if (tiles * ((p.M + 31) / 32) <= 256) return q4_run<T, SW, 1, 2, GPC>(p, st);
        return q4_run<T, SW, 2, 2, GPC>(p, st);
    } else if (p.M <= 16) {
        const int wide = (tiles > 256) + (tiles > 512) - (p.M <= 4);
        if (wide <= 0) return q4_run<T, SW, 1, 1, GPC>(p, st);
        return wide == 1 ? q4_run<T, SW, 2, 1, GPC>(p, st) : q4_run<T, SW, 4, 1, GPC>(p, st);
    } else {
        const int64_t work = tiles * ((p.M + 31) / 32);
        if (work <= 256) return q4_run<T, SW, 1, 2, GPC>(p, st);
        return work <= 512 ? q4_run<T, SW, 2, 2, GPC>(p, st) : q4_run<T, SW, 4, 2, GPC>(p, st);
    }
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
        // An odd K leaves half a byte, whatever it holds.
        const int half = bytes - 1 - at;
        if ((K & 1) && half >= 0 && half < 4) x &= ~(0xf0u << 8 * half);
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
    p.zeros = a->zeros ? a->zeros : a->scales;
    p.zero_mask = a->zeros ? ~0u : 0u;
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
    p.scale_bf16 = a->scale_dtype == TT_BF16 ? ~0u : 0u;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->dtype == TT_F32) return q4_typed<float>(a->scale_dtype, p, group < 128, st);
    if (a->dtype == TT_BF16) return q4_typed<__bf16>(a->scale_dtype, p, group < 128, st);
    return q4_typed<_Float16>(a->scale_dtype, p, group < 128, st);
}
