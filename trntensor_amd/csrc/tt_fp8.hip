// Products of rows in 8 bits with 8-bit weights (tt_fp8_matmul), and the gated
// half of a feed-forward block on two of them (tt_fp8_gated_matmul).
//
//   y[m][n] = sum_b sx[m][b] sw[n / 128][b] sum_{k in block b} cx[m][k] cw[n][k]
//
// The rows' scales are powers of two, which the scaled matrix instructions
// apply to what they sum; so are weights' of TT_E8M0. Floats multiply a block's
// sum on its way into the accumulators.
#include <type_traits>

#include "tt_fp8_block.hpp"

namespace tt {

namespace {

constexpr int kWaves = 8;

// A few rows: one workgroup of eight wavefronts R tiles of 16 weight rows (of
// either matrix where gated) and 16 rows of x. The wavefronts share the columns,
// four blocks of 128 in flight each, and their sums are joined in their order.
template <typename T, bool EXACT, bool E8, int R, bool GATED>
__global__ __launch_bounds__(64 * kWaves, 4) void fp8_rows_kernel(Fp8Params p) {
    constexpr int G = GATED ? 2 : 1, U = 4;
    __shared__ float so[kWaves][G * R][16][20];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const int tiles = (p.N + 15) / 16, row_blocks = (tiles + R - 1) / R, m_blocks = (p.M + 15) / 16;
    // Workgroup i runs on XCD i % 8: the blocks of x's rows that read the same
    // weights follow each other on one XCD, and share its L2.
    int rb, mb;
    const int tail = row_blocks % kNumXcd, even = (row_blocks - tail) * m_blocks;
    if ((int)blockIdx.x < even) {
        rb = blockIdx.x / (kNumXcd * m_blocks) * kNumXcd + blockIdx.x % kNumXcd;
        mb = blockIdx.x / kNumXcd % m_blocks;
    } else {
        rb = row_blocks - tail + (blockIdx.x - even) % tail;
        mb = (blockIdx.x - even) / tail;
    }
    const int m0 = mb * 16, per = (p.blocks + kWaves - 1) / kWaves;
    const int first = wave * per, last = first + per < p.blocks ? first + per : p.blocks;
    // Rows past the end repeat the last one: what they give is not stored.
    const int row = m0 + c < p.M ? m0 + c : p.M - 1;
    const uint8_t* x_row = p.x + (int64_t)row * p.blocks * 128 + g * 16;
    const uint8_t* s_row = p.xs + (int64_t)row * p.x_scales;
    const uint8_t* w_tile[G * R];
    int tile[G * R];
    f32x4 out[G * R];
#pragma unroll
    for (int r = 0; r < G * R; ++r) {
        tile[r] = rb * R + r / G < tiles ? rb * R + r / G : tiles - 1;
        w_tile[r] = p.w[r % G] + (int64_t)tile[r] * p.blocks * 2048 + lane * 16;
        out[r] = f32x4{0, 0, 0, 0};
    }
    // Loads of `many` blocks ahead of their products. (No condition among them:
    // the compiler would put each load behind it.)
    auto fold = [&](auto many, int k) __attribute__((always_inline)) {
        constexpr int V = decltype(many)::value;
        Block<EXACT, E8> a[V][G * R], b[V];
        uint32_t sa[V][G * R], sb;
#pragma unroll
        for (int u = 0; u < V; ++u) {
#pragma unroll
            for (int r = 0; r < G * R; ++r) {
                const uint8_t* w = w_tile[r] + (int64_t)(k + u) * 2048;
                a[u][r].load(w, w + 1024);
                sa[u][r] = weight_scale<E8>(p, r % G, tile[r], k + u);
            }
            b[u].load(x_row + (int64_t)(k + u) * 128, x_row + (int64_t)(k + u) * 128 + 64);
        }
        // Four scales of the row at once, from where it has four.
        const int from = k < p.x_scales - 4 ? k : p.x_scales - 4;
        __builtin_memcpy(&sb, s_row + from, 4);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < V; ++u)
#pragma unroll
            for (int r = 0; r < G * R; ++r) mma_block(a[u][r], b[u], out[r], sa[u][r], sb >> (k - from + u) * 8 & 255);
    };
    int k = first;
    for (; k + U <= last; k += U) fold(std::integral_constant<int, U>(), k);
    if (k + 2 <= last) {
        fold(std::integral_constant<int, 2>(), k);
        k += 2;
    }
    if (k < last) fold(std::integral_constant<int, 1>(), k);
#pragma unroll
    for (int r = 0; r < G * R; ++r) *reinterpret_cast<f32x4*>(&so[wave][r][c][g * 4]) = out[r];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * R * 4; i += 64 * kWaves) {
        const int m = i / (R * 4), r = i / 4 % R, n = i % 4 * 4;
        if (m0 + m >= p.M || (rb * R + r) * 16 + n >= p.N) continue;
        f32x4 v[G];
#pragma unroll
        for (int q = 0; q < G; ++q) {
            v[q] = *reinterpret_cast<const f32x4*>(&so[0][r * G + q][m][n]);
#pragma unroll
            for (int w = 1; w < kWaves; ++w) v[q] += *reinterpret_cast<const f32x4*>(&so[w][r * G + q][m][n]);
        }
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = GATED ? gate_value(v[0][j], v[G - 1][j], p.activation) : v[0][j];
        store_row(static_cast<T*>(p.y) + (int64_t)(m0 + m) * p.N, (rb * R + r) * 16 + n, p.N, y);
    }
}

template <bool EXACT, bool E8, int R, bool GATED>
int rows_run(int kind, const Fp8Params& p, hipStream_t st) {
    const int64_t grid = ((int64_t)(p.N + 15) / 16 + R - 1) / R * ((p.M + 15) / 16);
    if (grid > kMaxGrid / 2) return set_error(TT_UNSUPPORTED, "8-bit products: %lld workgroups", (long long)grid);
    // Results in 32 bits are exact sums or, of the gated block, what a second launch rounds.
    if constexpr (EXACT || GATED) {
        if (EXACT || kind == kRaw) {
            fp8_rows_kernel<float, EXACT, E8, R, GATED><<<(uint32_t)grid, 64 * kWaves, 0, st>>>(p);
            return check_launch("8-bit products");
        }
    }
    if constexpr (!EXACT) {
        if (p.bf16)
            fp8_rows_kernel<__bf16, EXACT, E8, R, GATED><<<(uint32_t)grid, 64 * kWaves, 0, st>>>(p);
        else
            fp8_rows_kernel<_Float16, EXACT, E8, R, GATED><<<(uint32_t)grid, 64 * kWaves, 0, st>>>(p);
    }
    return check_launch("8-bit products");
}

// Two weight tiles a workgroup from 512 workgroups on: 32 / 64 rows on 4096 x 4096
// take 6.5 / 9.1 us with two, 7.8 / 12.7 with one, 9.0 / 9.1 with four; 1 and 16
// rows (256 workgroups) 5.3 / 6.5 with two, 5.0 / 5.8 with one. Two blocks of x's
// rows a workgroup were slower for each (64 rows: 9.2 for 9.1 us, 128: 14.3 for 15.0).
bool two_tiles(const Fp8Params& p) { return (int64_t)((p.N + 15) / 16) * ((p.M + 15) / 16) >= 512 && p.M > 16; }

template <bool EXACT, bool E8, bool GATED>
int rows_shape(int kind, const Fp8Params& p, hipStream_t st) {
    if constexpr (!GATED)
        if (two_tiles(p)) return rows_run<EXACT, E8, 2, GATED>(kind, p, st);
    return rows_run<EXACT, E8, 1, GATED>(kind, p, st);
}

template <bool GATED>
int rows(int kind, bool e8, const Fp8Params& p, hipStream_t st) {
    if (kind == kExact) return e8 ? rows_shape<true, true, GATED>(kind, p, st) : rows_shape<true, false, GATED>(kind, p, st);
    return e8 ? rows_shape<false, true, GATED>(kind, p, st) : rows_shape<false, false, GATED>(kind, p, st);
}

// About how many us the workgroups above take: what they read at 17 TB/s (16 to
// 64 rows on 4096 x 4096, 60 on 1523 x 7009: 15 to 20).
double rows_cost(const Fp8Params& p, bool gated) {
    const int r = gated || two_tiles(p) ? 2 : 1;
    const double groups = (double)((p.N + 15) / 16) * (gated ? 2 : 1) / r * ((p.M + 15) / 16);
    return groups * p.blocks * (r * 2048 + (p.M < 16 ? p.M : 16) * 128) / 17e6;
}

// Offsets within a tile's rows are of 32 bits.
bool tiles_can(const Fp8Params& p) { return p.K <= 1 << 23; }

// us that a second launch and the float32 values between the two take: tiles that
// write codes / a second launch, M x N x K: 4 x 2816 x 1024 8.2 / 11.5, 100 x 2816
// x 2048 11.0 / 11.6, 500 x 2816 x 2048 15.3 / 18.9, 128 x 12288 x 4096 32.8 / 35.5,
// but 16 x 12288 x 4096 28.3 / 25.8, 183 x 2176 x 5888 24.3 / 20.8.
constexpr double kLaunch = 7.0;

// How a gated call into 8 bits goes: on tiles that write codes, or as 32-bit
// products (on other tiles, or on few rows' workgroups) that a second launch rounds.
struct GatedPlan {
    bool tiles, fused;
    int which;
};

GatedPlan gated_plan(const Fp8Params& p, int kind) {
    GatedPlan plan = {false, false, 0};
    if (!tiles_can(p)) return plan;
    int which = 0;
    double best = rows_cost(p, true);
    const double cost = fp8_gated_tiles_cost(p, kind == kCodes ? kRaw : kind, &which);
    if (cost < best) plan = {true, false, which}, best = cost;
    if (kind == kCodes) {
        const double fused = fp8_gated_tiles_cost(p, kCodes, &which) - kLaunch;
        if (fused < best) plan = {true, true, which};
    }
    return plan;
}

// One thread 16 bytes of a tile.
__global__ __launch_bounds__(256) void fp8_pack_kernel(int64_t N, int64_t K, int64_t blocks, const uint8_t* codes, int64_t pitch,
                                                       u32x4* out, int64_t count) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= count) return;
    const int l = i & 63, h = i >> 6 & 1;
    const int64_t tile = i >> 7;
    const int64_t n = tile / blocks * 16 + (l & 15), k = tile % blocks * 128 + 64 * h + 16 * (l >> 4);
    u32x4 v = {0, 0, 0, 0};
    if (n < N && k + 16 <= K) {
        __builtin_memcpy(&v, codes + n * pitch + k, 16);
    } else if (n < N) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (k + j < K) v[j / 4] |= (uint32_t)codes[n * pitch + k + j] << 8 * (j % 4);
    }
    out[i] = v;
}

int check_weights(const char* who, int64_t N, int64_t K) {
    constexpr int64_t kMost = int64_t(1) << 30;
    if (N < 0 || K < 1) return set_error(TT_INVALID, "%s: %lld rows of %lld columns", who, (long long)N, (long long)K);
    if (N > kMost || K > kMost) return set_error(TT_UNSUPPORTED, "%s: extents beyond 2^30", who);
    return TT_OK;
}

int check_product(const char* who, int64_t dtype, int64_t scale_dtype, int64_t M, int64_t N, int64_t K) {
    if (!serving_dtype(dtype)) return set_error(TT_UNSUPPORTED, "%s: dtype %lld (TT_F32, TT_BF16, TT_F16)", who, (long long)dtype);
    if (scale_dtype != TT_F32 && scale_dtype != TT_E8M0)
        return set_error(TT_UNSUPPORTED, "%s: scale dtype %lld (TT_F32, TT_E8M0)", who, (long long)scale_dtype);
    if (int rc = check_weights(who, N, K)) return rc;
    if (M < 0) return set_error(TT_INVALID, "%s: %lld rows", who, (long long)M);
    if (M > int64_t(1) << 30) return set_error(TT_UNSUPPORTED, "%s: extents beyond 2^30", who);
    return TT_OK;
}

Fp8Params params_of(int64_t M, int64_t N, int64_t K, const void* x, const void* xs) {
    Fp8Params p = {};
    p.x = static_cast<const uint8_t*>(x);
    p.xs = static_cast<const uint8_t*>(xs);
    p.M = (int)M;
    p.N = (int)N;
    p.K = (int)K;
    p.blocks = (int)fp8_blocks(K);
    p.x_scales = (int)fp8_scales(K);
    return p;
}

}  // namespace
}  // namespace tt

extern "C" size_t tt_fp8_packed_bytes(int64_t N, int64_t K) {
    if (N < 1 || K < 1) return 0;
    return (size_t)((N + 15) / 16) * (size_t)((K + 127) / 128) * 2048;
}

extern "C" int tt_fp8_pack(int64_t N, int64_t K, const void* codes, int64_t pitch, void* packed, void* stream) {
    using namespace tt;
    if (int rc = check_weights("tt_fp8_pack", N, K)) return rc;
    if (N == 0) return TT_OK;
    if (!codes || !packed) return set_error(TT_INVALID, "tt_fp8_pack: NULL pointer");
    if (pitch < K || (uintptr_t)packed % 16)
        return set_error(TT_INVALID, "tt_fp8_pack: pitch %lld, or alignment", (long long)pitch);
    const int64_t count = (int64_t)(tt_fp8_packed_bytes(N, K) / 16), grid = (count + 255) / 256;
    if (grid > kMaxGrid) return set_error(TT_UNSUPPORTED, "tt_fp8_pack: %lld by %lld codes", (long long)N, (long long)K);
    fp8_pack_kernel<<<(uint32_t)grid, 256, 0, static_cast<hipStream_t>(stream)>>>(
        N, K, fp8_blocks(K), static_cast<const uint8_t*>(codes), pitch, static_cast<u32x4*>(packed), count);
    return check_launch("tt_fp8_pack");
}

extern "C" int tt_fp8_matmul(const tt_fp8_matmul_args* a, void* stream) {
    using namespace tt;
    if (!a) return set_error(TT_INVALID, "tt_fp8_matmul: NULL arguments");
    if (int rc = check_product("tt_fp8_matmul", a->dtype, a->scale_dtype, a->M, a->N, a->K)) return rc;
    if (a->M == 0 || a->N == 0) return TT_OK;
    if (!a->x || !a->x_scales || !a->w || !a->w_scales || !a->y) return set_error(TT_INVALID, "tt_fp8_matmul: NULL pointer");
    if (((uintptr_t)a->x | (uintptr_t)a->w) % 16 || ((uintptr_t)a->x_scales | (uintptr_t)a->w_scales) % 4)
        return set_error(TT_INVALID, "tt_fp8_matmul: codes and scales are not aligned to 16 and 4 bytes");
    Fp8Params p = params_of(a->M, a->N, a->K, a->x, a->x_scales);
    p.w[0] = static_cast<const uint8_t*>(a->w);
    p.ws[0] = static_cast<const uint8_t*>(a->w_scales);
    p.y = a->y;
    p.bf16 = a->dtype == TT_BF16;
    const bool exact = a->dtype == TT_F32, e8 = a->scale_dtype == TT_E8M0;
    hipStream_t st = static_cast<hipStream_t>(stream);
    int which = 0;
    if (tiles_can(p) && fp8_tiles_cost(p, exact, &which) < rows_cost(p, false)) return fp8_tiles(exact, e8, which, p, st);
    return rows<false>(exact ? kExact : kHalf, e8, p, st);
}

extern "C" size_t tt_fp8_gated_workspace_bytes(const tt_fp8_gated_args* a) {
    using namespace tt;
    if (!a || !a->codes || a->M < 1 || a->N < 1 || a->K < 1 || a->M > 1 << 30 || a->N > 1 << 30 || a->K > 1 << 30) return 0;
    return gated_plan(params_of(a->M, a->N, a->K, nullptr, nullptr), kCodes).fused ? 0 : (size_t)a->M * (size_t)a->N * 4;
}

extern "C" int tt_fp8_gated_matmul(const tt_fp8_gated_args* a, void* stream) {
    using namespace tt;
    constexpr const char* who = "tt_fp8_gated_matmul";
    if (!a) return set_error(TT_INVALID, "%s: NULL arguments", who);
    if (int rc = check_product(who, a->dtype, a->scale_dtype, a->M, a->N, a->K)) return rc;
    if (a->activation != 0 && a->activation != 1) return set_error(TT_INVALID, "%s: activation %lld", who, (long long)a->activation);
    if (a->M == 0 || a->N == 0) return TT_OK;
    if (!a->x || !a->x_scales || !a->gate || !a->gate_scales || !a->up || !a->up_scales || !a->codes != !a->scales || !a->y == !a->codes)
        return set_error(TT_INVALID, "%s: NULL pointer, or both of y and codes", who);
    if (((uintptr_t)a->x | (uintptr_t)a->gate | (uintptr_t)a->up | (uintptr_t)a->codes) % 16 ||
        ((uintptr_t)a->x_scales | (uintptr_t)a->gate_scales | (uintptr_t)a->up_scales | (uintptr_t)a->scales | (uintptr_t)a->workspace) % 4)
        return set_error(TT_INVALID, "%s: codes and scales are not aligned to 16 and 4 bytes", who);
    const size_t need = tt_fp8_gated_workspace_bytes(a);
    if (need && (!a->workspace || a->workspace_bytes < (int64_t)need))
        return set_error(TT_INVALID, "%s: workspace of %lld bytes, %zu needed", who, (long long)a->workspace_bytes, need);
    Fp8Params p = params_of(a->M, a->N, a->K, a->x, a->x_scales);
    p.w[0] = static_cast<const uint8_t*>(a->gate);
    p.ws[0] = static_cast<const uint8_t*>(a->gate_scales);
    p.w[1] = static_cast<const uint8_t*>(a->up);
    p.ws[1] = static_cast<const uint8_t*>(a->up_scales);
    p.activation = (int)a->activation;
    p.codes = static_cast<uint8_t*>(a->codes);
    p.scales = static_cast<uint8_t*>(a->scales);
    p.bf16 = a->dtype == TT_BF16;
    const bool e8 = a->scale_dtype == TT_E8M0;
    const int kind = a->codes ? kCodes : a->dtype == TT_F32 ? kExact : kHalf;
    const GatedPlan plan = gated_plan(p, kind);
    p.y = a->codes ? a->workspace : a->y;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->codes && !plan.fused && a->M * ((a->N + 2047) / 2048) > kMaxGrid)
        return set_error(TT_UNSUPPORTED, "%s: %lld rows of %lld", who, (long long)a->M, (long long)a->N);
    if (plan.fused) return fp8_gated_tiles(kCodes, e8, plan.which, p, st);
    const int first = a->codes ? kRaw : kind;
    if (int rc = plan.tiles ? fp8_gated_tiles(first, e8, plan.which, p, st) : rows<true>(first, e8, p, st)) return rc;
    return a->codes ? fp8_gated_round(e8, p, st) : TT_OK;
}
