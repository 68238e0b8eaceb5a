// Rows into 8 bits (tt_fp8_quantize), and the root-mean-square norm with the
// residual stream's addition (tt_rms_norm):
//   h = x + residual,  y = h / sqrt(mean(h^2) + eps) * weight
#include <cmath>

#include "tt_fp8.hpp"

namespace tt {

namespace {

constexpr int kThreads = 256;

struct RowParams {
    const void *x, *residual, *weight;
    void *sum, *y;
    uint8_t *codes, *scales;
    int64_t x_stride, r_stride, rows;
    int dim, blocks;
    int weight_dtype;
    float eps, eps_root;
    double eps_exact;
};

__device__ __forceinline__ float wave_sum32(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
    return v;
}

__device__ __forceinline__ float wave_max32(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, kWave));
    return v;
}

// 2^-e of a positive float of exponent e (2^127 at most).
__device__ __forceinline__ float inverse_power(float x) {
    const uint32_t field = 254u - (__float_as_uint(x) >> 23);
    return __uint_as_float((field < 254u ? field : 254u) << 23);
}

// W: float, or __bf16 for weights of either 16-bit type. LANES lanes a row (a
// wavefront, or the workgroup), eight elements of it a pass. HBM bounds it: up to
// PASSES passes stay in registers, so that rows are read once, all loads of a row
// in flight, and 8192 rows of 8192 with the residual stream take 87 us where a copy
// of as many bytes takes 92. Longer rows (PASSES 0) are read again, from L2.
template <typename T, typename W, int LANES, int PASSES>
__global__ __launch_bounds__(kThreads) void rms_norm_kernel(RowParams p) {
    constexpr int STEP = LANES * 8, HELD = PASSES > 0 ? PASSES : 1;
    __shared__ float part[kThreads / kWave];
    const int64_t row = (int64_t)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
    if (row >= p.rows) return;  // whole wavefronts, and no barrier where a row is one
    const int first = threadIdx.x % LANES * 8;
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* r = p.residual ? static_cast<const T*>(p.residual) + row * p.r_stride : nullptr;
    const W* weight = static_cast<const W*>(p.weight);
    const int end = p.codes ? p.blocks * 128 : p.dim;
    auto total = [&](int col, float (&v)[8]) __attribute__((always_inline)) {
        Eight<T> a, b;
        a.load(x, col, p.dim);
        if (r) b.load(r, col, p.dim);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = r ? a.get(i) + b.get(i) : a.get(i);
    };
    float v[HELD][8], power = 0.f;
    Eight<W> w[HELD];
    // Of long rows the weights come once the sum is known: their registers would
    // halve the wavefronts that a CU holds (4096 rows of 16384: 122 us early, 94 so).
    constexpr bool EARLY = PASSES > 0 && PASSES <= 2;
    if constexpr (PASSES > 0) {
        Eight<T> a[PASSES], b[PASSES];
#pragma unroll
        for (int u = 0; u < PASSES; ++u) a[u].load(x, first + u * STEP, p.dim);
        if (r)
#pragma unroll
            for (int u = 0; u < PASSES; ++u) b[u].load(r, first + u * STEP, p.dim);
        if constexpr (EARLY)
#pragma unroll
            for (int u = 0; u < PASSES; ++u)
                if (p.weight) w[u].load(weight, first + u * STEP, p.dim);
#pragma unroll
        for (int u = 0; u < PASSES; ++u) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[u][i] = a[u].get(i);
            if (r) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[u][i] += b[u].get(i);
                store_row(static_cast<T*>(p.sum) + row * p.dim, first + u * STEP, p.dim, v[u]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) power += v[u][i] * v[u][i];
        }
    } else {
        for (int col = first; col < p.dim; col += STEP) {
            total(col, v[0]);
            if (r) store_row(static_cast<T*>(p.sum) + row * p.dim, col, p.dim, v[0]);
#pragma unroll
            for (int i = 0; i < 8; ++i) power += v[0][i] * v[0][i];
        }
    }
    // The wavefronts' sums or maxima of a row, in their order.
    auto joined = [&](float value, auto join) __attribute__((always_inline)) {
        if constexpr (LANES == kWave) return value;
        if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = value;
        __syncthreads();
        value = part[0];
#pragma unroll
        for (int i = 1; i < kThreads / kWave; ++i) value = join(value, part[i]);
        return value;
    };
    auto add = [](float a, float b) __attribute__((always_inline)) { return a + b; };
    float mean = joined(wave_sum32(power), add) / (float)p.dim + p.eps;
    // Squares of elements from 2^55 on may pass 2^128 in a row, and below 2^-50 lose bits or
    // vanish, which counts where eps is as small. Such rows (all lanes have one mean) are summed
    // again, times a power of two that brings the larger of their top and eps's root to 1.
    // From 2^63 on they stay as they are: zeros over an infinite mean.
    float lift = 1.f;
    if (!(mean >= 0x1p-100f && mean < INFINITY)) {
        auto each = [&](auto use) __attribute__((always_inline)) {
            if constexpr (PASSES > 0) {
#pragma unroll
                for (int u = 0; u < PASSES; ++u) use(v[u]);
            } else {
                for (int col = first; col < p.dim; col += STEP) {
                    total(col, v[0]);
                    use(v[0]);
                }
            }
        };
        float top = 0.f;
        each([&](const float (&h)[8]) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(h[i]));
        });
        if constexpr (LANES > kWave) __syncthreads();
        top = joined(wave_max32(top), [](float a, float b) __attribute__((always_inline)) { return fmaxf(a, b); });
        const float high = fmaxf(top, p.eps_root);
        if (high > 0.f && top < 0x1p63f) {
            lift = inverse_power(high);
            power = 0.f;
            each([&](float (&h)[8]) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) h[i] *= lift, power += h[i] * h[i];
            });
            if constexpr (LANES > kWave) __syncthreads();
            mean = joined(wave_sum32(power), add) / (float)p.dim + (float)(p.eps_exact * lift * lift);
        } else if (high == 0.f && p.eps_exact > 0.0) {
            mean = 1.f;  // zeros over an eps that is none in 32 bits
        }
    }
    const float scale = 1.f / sqrtf(mean);
    auto finish = [&](int col, float (&v)[8], const Eight<W>& w) __attribute__((always_inline)) {
        // Past the row's end these stay zeros, whatever the scale.
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = col + i < p.dim ? v[i] * scale : 0.f;
        if (p.weight)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= w.get(i, p.weight_dtype == TT_BF16);
        if (p.codes)
            fp8_store8(v, col, p.blocks, p.codes + row * p.blocks * 128, p.scales + row * ((p.blocks + 3) / 4 * 4));
        else
            store_row(static_cast<T*>(p.y) + row * p.dim, col, p.dim, v);
    };
    if constexpr (PASSES > 0) {
#pragma unroll
        for (int u = 0; u < PASSES; ++u)
            if (first + u * STEP < end) {
                if constexpr (!EARLY)
                    if (p.weight) w[u].load(weight, first + u * STEP, p.dim);
                finish(first + u * STEP, v[u], w[u]);
            }
    } else {
        for (int col = first; col < end; col += STEP) {
            if (p.weight) w[0].load(weight, col, p.dim);
            total(col, v[0]);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[0][i] *= lift;
            finish(col, v[0], w[0]);
        }
    }
}

// Workgroups: four rows each up to 1024 elements, else one.
int64_t rms_norm_grid(int64_t rows, int64_t dim) { return dim <= 1024 ? (rows + 3) / 4 : rows; }

template <typename T, typename W>
int rms_norm_run(const RowParams& p, hipStream_t st) {
    const uint32_t grid = (uint32_t)rms_norm_grid(p.rows, p.dim);
    if (p.dim <= 512)
        rms_norm_kernel<T, W, 64, 1><<<grid, kThreads, 0, st>>>(p);
    else if (p.dim <= 1024)
        rms_norm_kernel<T, W, 64, 2><<<grid, kThreads, 0, st>>>(p);
    else if (p.dim <= 2048)
        rms_norm_kernel<T, W, 256, 1><<<grid, kThreads, 0, st>>>(p);
    else if (p.dim <= 4096)
        rms_norm_kernel<T, W, 256, 2><<<grid, kThreads, 0, st>>>(p);
    else if (p.dim <= 8192)
        rms_norm_kernel<T, W, 256, 4><<<grid, kThreads, 0, st>>>(p);
    else if (p.dim <= 16384)
        rms_norm_kernel<T, W, 256, 8><<<grid, kThreads, 0, st>>>(p);
    else
        rms_norm_kernel<T, W, 256, 0><<<grid, kThreads, 0, st>>>(p);
    return check_launch("tt_rms_norm");
}

// `each` lanes a row, or workgroups of 2048 elements of one (`pieces` of them). What
// is written is half of what is read or less: 16384 rows of 8192 bfloat16 take 72
// us, 5.6 TB/s of reading and writing.
template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_kernel(RowParams p, int pieces, int each) {
    const int64_t row = pieces > 1 ? blockIdx.x / pieces : (int64_t)blockIdx.x * (kThreads / each) + threadIdx.x / each;
    if (row >= p.rows) return;
    const int col = (pieces > 1 ? (int)(blockIdx.x % pieces) * kThreads * 8 : 0) + (int)(threadIdx.x % each) * 8;
    Eight<T> x;
    x.load(static_cast<const T*>(p.x) + row * p.x_stride, col, p.dim);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x.get(i);
    fp8_store8(v, col, p.blocks, p.codes + row * p.blocks * 128, p.scales + row * ((p.blocks + 3) / 4 * 4));
}

template <typename T>
int quantize_run(const RowParams& p, hipStream_t st) {
    quantize_kernel<T><<<(uint32_t)fp8_quantize_grid(p.rows, p.dim), kThreads, 0, st>>>(p, (p.dim + 2047) / 2048, fp8_quantize_lanes(p.dim));
    return check_launch("tt_fp8_quantize");
}

int check_rows(const char* who, int64_t dtype, int64_t rows, int64_t dim) {
    constexpr int64_t kMost = int64_t(1) << 30;
    if (!serving_dtype(dtype)) return set_error(TT_UNSUPPORTED, "%s: dtype %lld (TT_F32, TT_BF16, TT_F16)", who, (long long)dtype);
    if (rows < 0 || dim < 1) return set_error(TT_INVALID, "%s: %lld rows of %lld", who, (long long)rows, (long long)dim);
    if (rows > kMost << 10 || dim > kMost) return set_error(TT_UNSUPPORTED, "%s: %lld rows of %lld", who, (long long)rows, (long long)dim);
    return TT_OK;
}

}  // namespace
}  // namespace tt

extern "C" int tt_rms_norm(const tt_rms_norm_args* a, void* stream) {
    using namespace tt;
    if (!a) return set_error(TT_INVALID, "tt_rms_norm: NULL arguments");
    if (int rc = check_rows("tt_rms_norm", a->dtype, a->rows, a->dim)) return rc;
    if (a->weight && !serving_dtype(a->weight_dtype))
        return set_error(TT_UNSUPPORTED, "tt_rms_norm: weight dtype %lld (TT_F32, TT_BF16, TT_F16)", (long long)a->weight_dtype);
    if (!(a->eps >= 0.0) || a->eps > 1e38) return set_error(TT_INVALID, "tt_rms_norm: eps %g", a->eps);
    if (rms_norm_grid(a->rows, a->dim) > kMaxGrid)
        return set_error(TT_UNSUPPORTED, "tt_rms_norm: %lld rows of %lld", (long long)a->rows, (long long)a->dim);
    if (a->rows == 0) return TT_OK;
    if (!a->x || !a->residual != !a->sum || !a->codes != !a->scales || !a->y == !a->codes)
        return set_error(TT_INVALID, "tt_rms_norm: NULL pointer, or both of y and codes");
    if ((uintptr_t)a->codes % 16 || (uintptr_t)a->scales % 4)
        return set_error(TT_INVALID, "tt_rms_norm: codes and scales are not aligned to 16 and 4 bytes");
    RowParams p = {};
    p.x = a->x;
    p.residual = a->residual;
    p.weight = a->weight;
    p.sum = a->sum;
    p.y = a->y;
    p.codes = static_cast<uint8_t*>(a->codes);
    p.scales = static_cast<uint8_t*>(a->scales);
    p.x_stride = a->x_stride;
    p.r_stride = a->residual_stride;
    p.dim = (int)a->dim;
    p.blocks = (int)fp8_blocks(a->dim);
    p.rows = a->rows;
    p.weight_dtype = (int)a->weight_dtype;
    p.eps = (float)a->eps;
    p.eps_root = (float)std::sqrt(a->eps);
    p.eps_exact = a->eps;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool wide = a->weight && a->weight_dtype == TT_F32;
    if (a->dtype == TT_F32) return wide ? rms_norm_run<float, float>(p, st) : rms_norm_run<float, __bf16>(p, st);
    if (a->dtype == TT_BF16) return wide ? rms_norm_run<__bf16, float>(p, st) : rms_norm_run<__bf16, __bf16>(p, st);
    return wide ? rms_norm_run<_Float16, float>(p, st) : rms_norm_run<_Float16, __bf16>(p, st);
}

extern "C" int tt_fp8_quantize(const tt_fp8_quantize_args* a, void* stream) {
    using namespace tt;
    if (!a) return set_error(TT_INVALID, "tt_fp8_quantize: NULL arguments");
    if (int rc = check_rows("tt_fp8_quantize", a->dtype, a->rows, a->dim)) return rc;
    if (fp8_quantize_grid(a->rows, a->dim) > kMaxGrid)
        return set_error(TT_UNSUPPORTED, "tt_fp8_quantize: %lld rows of %lld", (long long)a->rows, (long long)a->dim);
    if (a->rows == 0) return TT_OK;
    if (!a->x || !a->codes || !a->scales) return set_error(TT_INVALID, "tt_fp8_quantize: NULL pointer");
    if ((uintptr_t)a->codes % 16 || (uintptr_t)a->scales % 4)
        return set_error(TT_INVALID, "tt_fp8_quantize: codes and scales are not aligned to 16 and 4 bytes");
    RowParams p = {};
    p.x = a->x;
    p.codes = static_cast<uint8_t*>(a->codes);
    p.scales = static_cast<uint8_t*>(a->scales);
    p.x_stride = a->x_stride;
    p.dim = (int)a->dim;
    p.blocks = (int)fp8_blocks(a->dim);
    p.rows = a->rows;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->dtype == TT_F32) return quantize_run<float>(p, st);
    return a->dtype == TT_BF16 ? quantize_run<__bf16>(p, st) : quantize_run<_Float16>(p, st);
}
