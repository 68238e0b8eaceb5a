// Products with 4-bit weights: y[m][n] = sum_k x[m][k] s[k/g][n] (c[n][k] - z[k/g][n]).
#include "tt_serving.hpp"

namespace tt {

namespace {

struct Q4Params {
    int64_t M, N, K, group, ldx, code_pitch, ldy;
    const void *x, *scales, *zeros;
    const uint8_t* codes;
    void* y;
};

template <typename S>
__device__ __forceinline__ float q4_zero(const Q4Params& p, int64_t i) {
    return p.zeros ? to_f32(static_cast<const S*>(p.zeros)[i]) : 8.f;
}

// One wavefront per output: each lane sums every 64th byte (two codes) of the row.
template <typename T, typename S>
__global__ __launch_bounds__(256) void q4_simple_kernel(Q4Params p) {
    const int lane = threadIdx.x & 63;
    const int64_t w = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
    if (w >= p.M * p.N) return;
    const int64_t n = w % p.N, m = w / p.N;
    const T* x = static_cast<const T*>(p.x) + m * p.ldx;
    const uint8_t* c = p.codes + n * p.code_pitch;
    float sum = 0.f;
    for (int64_t j = lane; 2 * j < p.K; j += 64) {
        const int64_t g = 2 * j / p.group * p.N + n;
        const float s = to_f32(static_cast<const S*>(p.scales)[g]), z = q4_zero<S>(p, g);
        const int byte = c[j];
        float part = to_f32(x[2 * j]) * ((float)(byte & 15) - z);
        if (2 * j + 1 < p.K) part += to_f32(x[2 * j + 1]) * ((float)(byte >> 4) - z);
        sum += s * part;
    }
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if (lane == 0) static_cast<T*>(p.y)[m * p.ldy + n] = (T)sum;
}

template <typename T, typename S>
int q4_launch(const Q4Params& p, hipStream_t st) {
    const int64_t blocks = (p.M * p.N + 3) / 4;
    if (blocks > kMaxGrid) return set_error(TT_UNSUPPORTED, "tt_q4_matmul: %lld outputs", (long long)(p.M * p.N));
    q4_simple_kernel<T, S><<<(uint32_t)blocks, 256, 0, st>>>(p);
    return check_launch("tt_q4_matmul");
}

template <typename T>
int q4_typed(int64_t scale_dtype, const Q4Params& p, hipStream_t st) {
    if (scale_dtype == TT_F32) return q4_launch<T, float>(p, st);
    if (scale_dtype == TT_BF16) return q4_launch<T, __bf16>(p, st);
    return q4_launch<T, _Float16>(p, st);
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
    if (a->M < 0 || a->N < 0 || a->K < 0) return set_error(TT_INVALID, "tt_q4_matmul: negative extent");
    if (a->group != 32 && a->group != 64 && (a->group < 128 || a->group % 128))
        return set_error(TT_INVALID, "tt_q4_matmul: group of %lld (32, 64 or a multiple of 128)", (long long)a->group);
    if (a->M == 0 || a->N == 0) return TT_OK;
    if (!a->y || (a->K > 0 && (!a->x || !a->codes || !a->scales)))
        return set_error(TT_INVALID, "tt_q4_matmul: NULL pointer");
    if (a->ldx < a->K || a->ldy < a->N) return set_error(TT_INVALID, "tt_q4_matmul: leading dimension below the width");
    if (a->code_pitch % 64 || a->code_pitch < (a->K + 1) / 2 || (uintptr_t)a->codes % 16)
        return set_error(TT_INVALID, "tt_q4_matmul: code pitch %lld or alignment", (long long)a->code_pitch);
    Q4Params p = {a->M,      a->N,        a->K,         a->group,    a->ldx,
                  a->code_pitch, a->ldy, a->x, a->scales, a->zeros, static_cast<const uint8_t*>(a->codes), a->y};
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->dtype == TT_F32) return q4_typed<float>(a->scale_dtype, p, st);
    if (a->dtype == TT_BF16) return q4_typed<__bf16>(a->scale_dtype, p, st);
    return q4_typed<_Float16>(a->scale_dtype, p, st);
}
