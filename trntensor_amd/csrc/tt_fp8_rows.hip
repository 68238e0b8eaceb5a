// Rows into 8 bits (tt_fp8_quantize), and the root-mean-square norm with the
// residual stream's addition (tt_rms_norm):
//   h = x + residual,  y = h / sqrt(mean(h^2) + eps) * weight
#include "tt_fp8.hpp"

namespace tt {

namespace {

constexpr int kThreads = 256;

struct RowParams {
    const void *x, *residual, *weight;
    void *sum, *y;
    uint8_t *codes, *scales;
    int64_t x_stride, r_stride, dim, blocks;
    int64_t rows;
    int weight_dtype;
    float eps;
};

__device__ __forceinline__ void load_weight(const RowParams& p, int64_t col, float (&w)[8]) {
    if (!p.weight) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 1.f;
    } else if (p.weight_dtype == TT_F32) {
        load_row(static_cast<const float*>(p.weight), col, p.dim, w);
    } else if (p.weight_dtype == TT_BF16) {
        load_row(static_cast<const __bf16*>(p.weight), col, p.dim, w);
    } else {
        load_row(static_cast<const _Float16*>(p.weight), col, p.dim, w);
    }
}

__device__ __forceinline__ float wave_sum32(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
    return v;
}

// One workgroup a row.
template <typename T>
__global__ __launch_bounds__(kThreads) void rms_norm_kernel(RowParams p) {
    __shared__ float part[kThreads / kWave];
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* r = p.residual ? static_cast<const T*>(p.residual) + row * p.r_stride : nullptr;
    auto load = [&](int64_t col, float (&v)[8]) {
        load_row(x, col, p.dim, v);
        if (r) {
            float a[8];
            load_row(r, col, p.dim, a);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += a[i];
        }
    };
    float power = 0.f;
    for (int64_t col = threadIdx.x * 8; col < p.dim; col += kThreads * 8) {
        float v[8];
        load(col, v);
        if (r) store_row(static_cast<T*>(p.sum) + row * p.dim, col, p.dim, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) power += v[i] * v[i];
    }
    power = wave_sum32(power);
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = power;
    __syncthreads();
    power = 0.f;
#pragma unroll
    for (int i = 0; i < kThreads / kWave; ++i) power += part[i];
    const float scale = 1.f / sqrtf(power / (float)p.dim + p.eps);
    const int64_t end = p.codes ? (p.blocks + 3) / 4 * 512 : p.dim;
    for (int64_t col = threadIdx.x * 8; col < end; col += kThreads * 8) {
        float v[8], w[8];
        load(col, v);
        load_weight(p, col, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = col + i < p.dim ? v[i] * scale * w[i] : 0.f;
        if (p.codes)
            fp8_store8(v, col, p.blocks, p.codes + row * p.blocks * 128, p.scales + row * ((p.blocks + 3) / 4 * 4));
        else
            store_row(static_cast<T*>(p.y) + row * p.dim, col, p.dim, v);
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_kernel(RowParams p) {
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    for (int64_t col = threadIdx.x * 8; col < (p.blocks + 3) / 4 * 512; col += kThreads * 8) {
        float v[8];
        load_row(x, col, p.dim, v);
        fp8_store8(v, col, p.blocks, p.codes + row * p.blocks * 128, p.scales + row * ((p.blocks + 3) / 4 * 4));
    }
}

int check_rows(const char* who, int64_t dtype, int64_t rows, int64_t dim) {
    constexpr int64_t kMost = int64_t(1) << 30;
    if (!serving_dtype(dtype)) return set_error(TT_UNSUPPORTED, "%s: dtype %lld (TT_F32, TT_BF16, TT_F16)", who, (long long)dtype);
    if (rows < 0 || dim < 1) return set_error(TT_INVALID, "%s: %lld rows of %lld", who, (long long)rows, (long long)dim);
    if (rows > kMaxGrid || dim > kMost) return set_error(TT_UNSUPPORTED, "%s: %lld rows of %lld", who, (long long)rows, (long long)dim);
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
    p.dim = a->dim;
    p.blocks = fp8_blocks(a->dim);
    p.rows = a->rows;
    p.weight_dtype = (int)a->weight_dtype;
    p.eps = (float)a->eps;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->dtype == TT_F32)
        rms_norm_kernel<float><<<(uint32_t)a->rows, kThreads, 0, st>>>(p);
    else if (a->dtype == TT_BF16)
        rms_norm_kernel<__bf16><<<(uint32_t)a->rows, kThreads, 0, st>>>(p);
    else
        rms_norm_kernel<_Float16><<<(uint32_t)a->rows, kThreads, 0, st>>>(p);
    return check_launch("tt_rms_norm");
}

extern "C" int tt_fp8_quantize(const tt_fp8_quantize_args* a, void* stream) {
    using namespace tt;
    if (!a) return set_error(TT_INVALID, "tt_fp8_quantize: NULL arguments");
    if (int rc = check_rows("tt_fp8_quantize", a->dtype, a->rows, a->dim)) return rc;
    if (a->rows == 0) return TT_OK;
    if (!a->x || !a->codes || !a->scales) return set_error(TT_INVALID, "tt_fp8_quantize: NULL pointer");
    if ((uintptr_t)a->codes % 16 || (uintptr_t)a->scales % 4)
        return set_error(TT_INVALID, "tt_fp8_quantize: codes and scales are not aligned to 16 and 4 bytes");
    RowParams p = {};
    p.x = a->x;
    p.codes = static_cast<uint8_t*>(a->codes);
    p.scales = static_cast<uint8_t*>(a->scales);
    p.x_stride = a->x_stride;
    p.dim = a->dim;
    p.blocks = fp8_blocks(a->dim);
    p.rows = a->rows;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->dtype == TT_F32)
        quantize_kernel<float><<<(uint32_t)a->rows, kThreads, 0, st>>>(p);
    else if (a->dtype == TT_BF16)
        quantize_kernel<__bf16><<<(uint32_t)a->rows, kThreads, 0, st>>>(p);
    else
        quantize_kernel<_Float16><<<(uint32_t)a->rows, kThreads, 0, st>>>(p);
    return check_launch("tt_fp8_quantize");
}
