// Appending keys and values to a paged cache of 8-bit floats, with the
// position rotation of keys and queries on the way.
#include "tt_serving.hpp"

namespace tt {

namespace {

struct AppendParams {
    int64_t tokens, q_heads, rot, interleaved, table_width, table_stride;
    int64_t k_stride[3], v_stride[3], q_stride[3];
    const void *k, *v, *q;
    void* q_out;
    const float *cos, *sin;
    const int32_t *table, *lengths, *counts;
    tt_kv_cache c;
    int64_t width, blocks;  // codes a row; blocks a sequence's new tokens may touch
    int64_t kv_groups;      // workgroups of the cache part; the rest rotate queries
};

// Element d of a row at position pos, rotated if d < rot. Products and sums
// are rounded one by one, as elementary operations round them.
template <typename T>
__device__ __forceinline__ float rotated(const AppendParams& p, const T* row, int64_t pos, int d) {
#pragma clang fp contract(off)
    const float x = to_f32(row[d]);
    if (!p.cos || d >= p.rot) return x;
    const int half = (int)p.rot / 2;
    const int pair = p.interleaved ? d / 2 : d % half;
    const bool second = p.interleaved ? d & 1 : d >= half;
    const float c = p.cos[pos * half + pair], s = p.sin[pos * half + pair];
    const int other = p.interleaved ? d ^ 1 : (second ? d - half : d + half);
    const float y = to_f32(row[other]);
    const float xc = x * c, ys = y * s;
    return second ? xc + ys : xc - ys;
}

// The smallest e with amax <= 448 * 2^e, at least -64: amax = 1.m * 2^u and 448 = 1.75 * 2^8.
__device__ __forceinline__ int scale_exponent(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -64 ? -64 : e;
}

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

template <typename T>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendParams p) {
    __shared__ float part[4];
    int64_t w = blockIdx.x;
    const int64_t H = p.c.heads, P = p.c.page, W = p.width;
    if (w >= p.kv_groups) {
        // queries: one workgroup per token
        w -= p.kv_groups;
        const int64_t b = w / p.tokens, t = w % p.tokens;
        const int64_t n = p.counts ? p.counts[b] : p.tokens, pos = (int64_t)p.lengths[b] + t;
        const bool live = t < n && pos >= 0 && pos < p.table_width * P;
        const T* q = static_cast<const T*>(p.q) + b * p.q_stride[0] + t * p.q_stride[1];
        T* out = static_cast<T*>(p.q_out) + w * p.q_heads * p.c.dim;
        for (int64_t i = threadIdx.x; i < p.q_heads * p.c.dim; i += 256) {
            const int64_t h = i / p.c.dim;
            out[i] = live ? (T)rotated<T>(p, q + h * p.q_stride[2], pos, (int)(i - h * p.c.dim)) : (T)0.f;
        }
        return;
    }
    const bool is_v = w & 1;
    w >>= 1;
    const int64_t j = w % p.blocks, h = w / p.blocks % H, b = w / p.blocks / H;
    const int64_t len = p.lengths[b];
    int64_t n = p.counts ? p.counts[b] : p.tokens;
    n = n > p.tokens ? p.tokens : n;
    if (len < 0) return;
    const int64_t end = len + n < p.table_width * P ? len + n : p.table_width * P;
    const int64_t first = (len / P + j) * P;
    const int64_t lo = (len > first ? len : first) - first, hi = (end < first + P ? end : first + P) - first;
    if (lo >= hi) return;
    const int64_t page = p.table[b * p.table_stride + first / P];
    if (page < 0 || page >= p.c.pages) return;
    const int64_t* stride = is_v ? p.v_stride : p.k_stride;
    const T* x = static_cast<const T*>(is_v ? p.v : p.k) + b * stride[0] + h * stride[2] + (first - len) * stride[1];
    uint8_t* codes = static_cast<uint8_t*>(is_v ? p.c.v : p.c.k) + (page * H + h) * W * P;
    float* scales = (is_v ? p.c.v_scale : p.c.k_scale) + page * H + h;
    auto value = [&](int64_t t, int d) -> float {
        if (d >= p.c.dim) return 0.f;
        return is_v ? to_f32(x[t * stride[1] + d]) : rotated<T>(p, x + t * stride[1], first + t, d);
    };
    auto place = [&](int64_t t, int64_t d) { return is_v ? d * P + t : t * W + d; };

    float amax = 0.f;
    for (int64_t i = lo * W + threadIdx.x; i < hi * W; i += 256) {
        const float a = fabsf(value(i / W, (int)(i % W)));
        if (a < INFINITY) amax = fmaxf(amax, a);
    }
    for (int off = 32; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off, 64));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x / 64] = amax;
    const float old = lo > 0 ? *scales : 0.f;
    __syncthreads();
    amax = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    const float scale = fmaxf(power_of_two(scale_exponent(amax)), old);
    const float inv = 1.f / scale;
    if (lo > 0 && scale > old) {
        for (int64_t i = threadIdx.x; i < lo * W; i += 256) {
            uint8_t* c = codes + place(i / W, i % W);
            *c = (uint8_t)fp8_pair(fp8_value(*c) * (old * inv), 0.f);
        }
    }
    for (int64_t i = lo * W + threadIdx.x; i < hi * W; i += 256) {
        const int64_t t = i / W, d = i % W;
        codes[place(t, d)] = (uint8_t)fp8_pair(value(t, (int)d) * inv, 0.f);
    }
    if (threadIdx.x == 0) *scales = scale;
}

template <typename T>
int append_launch(const AppendParams& p, int64_t grid, hipStream_t st) {
    kv_append_kernel<T><<<(uint32_t)grid, 256, 0, st>>>(p);
    return check_launch("tt_kv_append");
}

}  // namespace
}  // namespace tt

extern "C" int tt_kv_append(const tt_kv_append_args* a, void* stream) {
    using namespace tt;
    if (!a) return set_error(TT_INVALID, "tt_kv_append: NULL arguments");
    if (!serving_dtype(a->dtype))
        return set_error(TT_UNSUPPORTED, "tt_kv_append: dtype %lld (TT_F32, TT_BF16, TT_F16)", (long long)a->dtype);
    if (int rc = check_cache("tt_kv_append", a->cache)) return rc;
    if (a->batch < 0 || a->tokens < 0 || a->q_heads < 0 || a->table_width < 0)
        return set_error(TT_INVALID, "tt_kv_append: negative extent");
    if (a->cos && (!a->sin || a->rot < 2 || a->rot % 2 || a->rot > a->cache.dim))
        return set_error(TT_INVALID, "tt_kv_append: %lld rotated elements of %lld", (long long)a->rot,
                         (long long)a->cache.dim);
    if (a->q && (!a->cos || !a->q_out || a->q_heads < 1))
        return set_error(TT_INVALID, "tt_kv_append: queries without cos and sin, q_out or heads");
    if (a->batch == 0 || a->tokens == 0) return TT_OK;
    if (!a->k || !a->v || !a->lengths || (a->table_width > 0 && !a->table))
        return set_error(TT_INVALID, "tt_kv_append: NULL pointer");
    AppendParams p;
    p.tokens = a->tokens;
    p.q_heads = a->q_heads;
    p.rot = a->rot;
    p.interleaved = a->interleaved;
    p.table_width = a->table_width;
    p.table_stride = a->table_stride;
    for (int i = 0; i < 3; ++i) {
        p.k_stride[i] = a->k_stride[i];
        p.v_stride[i] = a->v_stride[i];
        p.q_stride[i] = a->q_stride[i];
    }
    p.k = a->k;
    p.v = a->v;
    p.q = a->q;
    p.q_out = a->q_out;
    p.cos = a->cos;
    p.sin = a->sin;
    p.table = a->table;
    p.lengths = a->lengths;
    p.counts = a->counts;
    p.c = a->cache;
    p.width = kv_width(a->cache.dim);
    p.blocks = (a->tokens + a->cache.page - 2) / a->cache.page + 1;
    p.kv_groups = 2 * a->batch * a->cache.heads * p.blocks;
    const int64_t grid = p.kv_groups + (a->q ? a->batch * a->tokens : 0);
    if (grid > kMaxGrid) return set_error(TT_UNSUPPORTED, "tt_kv_append: %lld workgroups", (long long)grid);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->dtype == TT_F32) return append_launch<float>(p, grid, st);
    if (a->dtype == TT_BF16) return append_launch<__bf16>(p, grid, st);
    return append_launch<_Float16>(p, grid, st);
}
