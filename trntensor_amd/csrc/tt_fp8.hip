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

// One workgroup of eight wavefronts a tile of 16 weight rows (two tiles where
// gated) and 16 MT rows of x; the wavefronts share the columns, and their sums
// are joined in their order.
template <typename T, bool EXACT, bool E8, int MT, bool GATED>
__global__ __launch_bounds__(64 * kWaves) void fp8_rows_kernel(Fp8Params p) {
    constexpr int R = GATED ? 2 : 1;
    __shared__ float so[kWaves][R][MT * 16][20];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const int tiles = (p.N + 15) / 16;
    const int tile = blockIdx.x % tiles, m0 = blockIdx.x / tiles * 16 * MT;
    const int per = (p.blocks + kWaves - 1) / kWaves;
    const int first = wave * per, last = first + per < p.blocks ? first + per : p.blocks;
    const uint8_t *x_row[MT], *s_row[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        // Rows past the end repeat the last one: what they give is not stored.
        const int m = m0 + mt * 16 + c < p.M ? m0 + mt * 16 + c : p.M - 1;
        x_row[mt] = p.x + (int64_t)m * p.blocks * 128 + g * 16;
        s_row[mt] = p.xs + (int64_t)m * p.x_scales;
    }
    f32x4 out[R][MT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) out[r][mt] = f32x4{0, 0, 0, 0};
    for (int k = first; k < last; ++k) {
        Block<EXACT, E8> b[MT];
        uint32_t sb[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            b[mt].load(x_row[mt] + (int64_t)k * 128, x_row[mt] + (int64_t)k * 128 + 64);
            sb[mt] = s_row[mt][k];
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint8_t* src = p.w[r] + ((int64_t)tile * p.blocks + k) * 2048 + lane * 16;
            Block<EXACT, E8> a;
            a.load(src, src + 1024);
            const uint32_t sa = weight_scale<E8>(p, r, tile, k);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) mma_block(a, b[mt], out[r][mt], sa, sb[mt]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) *reinterpret_cast<f32x4*>(&so[wave][r][mt * 16 + c][g * 4]) = out[r][mt];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * 16 * 4; i += 64 * kWaves) {
        const int m = i / 4, n = i % 4 * 4;
        if (m0 + m >= p.M || tile * 16 + n >= p.N) continue;
        f32x4 v[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            v[r] = *reinterpret_cast<const f32x4*>(&so[0][r][m][n]);
#pragma unroll
            for (int w = 1; w < kWaves; ++w) v[r] += *reinterpret_cast<const f32x4*>(&so[w][r][m][n]);
        }
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = GATED ? gate_value(v[0][j], v[R - 1][j], p.activation) : v[0][j];
        store_row(static_cast<T*>(p.y) + (int64_t)(m0 + m) * p.N, tile * 16 + n, p.N, y);
    }
}

template <typename T, bool EXACT, bool E8, bool GATED>
int fp8_rows(const Fp8Params& p, hipStream_t st) {
    const int64_t tiles = (p.N + 15) / 16;
    const int mt = p.M <= 16 ? 1 : 2;
    const int64_t grid = tiles * ((p.M + 16 * mt - 1) / (16 * mt));
    if (grid > kMaxGrid / 2) return set_error(TT_UNSUPPORTED, "8-bit products: %lld workgroups", (long long)grid);
    if (mt == 1)
        fp8_rows_kernel<T, EXACT, E8, 1, GATED><<<(uint32_t)grid, 64 * kWaves, 0, st>>>(p);
    else
        fp8_rows_kernel<T, EXACT, E8, 2, GATED><<<(uint32_t)grid, 64 * kWaves, 0, st>>>(p);
    return check_launch("8-bit products");
}

template <bool E8, bool GATED>
int fp8_typed(int64_t dtype, const Fp8Params& p, hipStream_t st) {
    if (GATED && p.codes) return fp8_rows<float, false, E8, GATED>(p, st);
    if (dtype == TT_F32) return fp8_rows<float, true, E8, GATED>(p, st);
    return dtype == TT_BF16 ? fp8_rows<__bf16, false, E8, GATED>(p, st) : fp8_rows<_Float16, false, E8, GATED>(p, st);
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

// Whether a call runs on workgroup tiles. (Their offsets within 256 rows are of 32 bits.)
bool many_rows_of(int64_t M, int64_t K) { return M >= 128 && K <= 1 << 23; }
bool many_rows(const Fp8Params& p) { return many_rows_of(p.M, p.K); }

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
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (many_rows(p)) return fp8_tiles(a->dtype, a->scale_dtype == TT_E8M0, false, p, st);
    return a->scale_dtype == TT_E8M0 ? fp8_typed<true, false>(a->dtype, p, st) : fp8_typed<false, false>(a->dtype, p, st);
}

extern "C" size_t tt_fp8_gated_workspace_bytes(const tt_fp8_gated_args* a) {
    using namespace tt;
    if (!a || !a->codes || a->M < 1 || a->N < 1 || a->K < 1 || many_rows_of(a->M, a->K)) return 0;
    return (size_t)a->M * (size_t)a->N * 4;
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
    hipStream_t st = static_cast<hipStream_t>(stream);
    p.codes = static_cast<uint8_t*>(a->codes);
    p.scales = static_cast<uint8_t*>(a->scales);
    p.y = a->y;
    if (many_rows(p)) return fp8_tiles(a->dtype, a->scale_dtype == TT_E8M0, true, p, st);
    if (a->codes) p.y = a->workspace;
    if (int rc = a->scale_dtype == TT_E8M0 ? fp8_typed<true, true>(a->dtype, p, st) : fp8_typed<false, true>(a->dtype, p, st)) return rc;
    if (!a->codes) return TT_OK;
    const tt_fp8_quantize_args q = {TT_F32, a->M, a->N, a->N, a->workspace, a->codes, a->scales};
    return tt_fp8_quantize(&q, stream);
}
