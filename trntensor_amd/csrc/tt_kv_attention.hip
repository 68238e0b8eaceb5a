// Attention over a paged cache of 8-bit floats.
#include "tt_serving.hpp"

namespace tt {

namespace {

struct AttnParams {
    int64_t tokens, q_heads, window, sinks, table_width, table_stride, q_stride[3];
    float scale;
    const void* q;
    void* out;
    const int32_t *table, *lengths, *counts;
    tt_kv_cache c;
    int64_t width;
};

// One workgroup per query row: chunks of 256 keys, running maximum and sum.
template <typename T>
__global__ __launch_bounds__(256) void kv_attention_simple_kernel(AttnParams p) {
    __shared__ float q[256], prob[256], part[4];
    const int tid = threadIdx.x;
    const int64_t H = p.c.heads, P = p.c.page, W = p.width, D = p.c.dim;
    const int64_t h = blockIdx.x % p.q_heads, t = blockIdx.x / p.q_heads % p.tokens, b = blockIdx.x / p.q_heads / p.tokens;
    const int64_t kh = h / (p.q_heads / H);
    T* out = static_cast<T*>(p.out) + blockIdx.x * D;
    int64_t len = p.lengths[b], n = p.counts ? p.counts[b] : p.tokens;
    const int64_t pos = len - n + t;
    if (len > p.table_width * P) len = p.table_width * P;
    const bool live = t < n && pos >= 0;
    const int64_t end = live ? (pos + 1 < len ? pos + 1 : len) : 0;  // keys [0, end)
    const int64_t low = p.window > 0 ? pos - p.window + 1 : 0;        // and of them [low, ..) or [0, sinks)
    const T* qrow = static_cast<const T*>(p.q) + b * p.q_stride[0] + t * p.q_stride[1] + h * p.q_stride[2];
    if (tid < D) q[tid] = to_f32(qrow[tid]);
    float top = -INFINITY, sum = 0.f, acc = 0.f;
    bool any = false;
    for (int64_t base = 0; base < end; base += 256) {
        if (base + 256 <= low && base >= p.sinks) continue;
        __syncthreads();
        const int64_t j = base + tid;
        float s = -INFINITY;
        bool seen = j < end && (j >= low || j < p.sinks);
        if (seen) {
            const int64_t page = p.table[b * p.table_stride + j / P];
            seen = page >= 0 && page < p.c.pages;
            if (seen) {
                const uint8_t* k = static_cast<const uint8_t*>(p.c.k) + ((page * H + kh) * P + j % P) * W;
                s = 0.f;
                for (int64_t d = 0; d < D; ++d) s += q[d] * fp8_value(k[d]);
                s *= p.c.k_scale[page * H + kh] * p.scale;
            }
        }
        float m = s;
        for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
        if ((tid & 63) == 0) part[tid / 64] = m;
        any = __syncthreads_or(seen) || any;
        m = fmaxf(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])), top);
        const float shift = m == -INFINITY ? 0.f : m;
        const float keep = expf(top - shift);
        const float e = seen ? expf(s - shift) : 0.f;
        prob[tid] = seen ? e : -1.f;
        sum = sum * keep + e;  // this thread's keys
        acc *= keep;
        top = m;
        __syncthreads();
        if (tid < D) {
            for (int i = 0; i < 256 && base + i < end; ++i) {
                if (prob[i] == -1.f) continue;
                const int64_t jj = base + i, page = p.table[b * p.table_stride + jj / P];
                const uint8_t* v = static_cast<const uint8_t*>(p.c.v) + ((page * H + kh) * W + tid) * P;
                acc += prob[i] * (fp8_value(v[jj % P]) * p.c.v_scale[page * H + kh]);
            }
        }
    }
    __syncthreads();
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if ((tid & 63) == 0) part[tid / 64] = sum;
    __syncthreads();
    sum = (part[0] + part[1]) + (part[2] + part[3]);
    if (tid < D) out[tid] = (T)(any ? acc / sum : 0.f);
}

template <typename T>
int attn_launch(const AttnParams& p, int64_t rows, hipStream_t st) {
    if (rows > kMaxGrid) return set_error(TT_UNSUPPORTED, "tt_kv_attention: %lld query rows", (long long)rows);
    kv_attention_simple_kernel<T><<<(uint32_t)rows, 256, 0, st>>>(p);
    return check_launch("tt_kv_attention");
}

int check_attention(const tt_kv_attention_args* a) {
    if (!a) return set_error(TT_INVALID, "tt_kv_attention: NULL arguments");
    if (!serving_dtype(a->dtype))
        return set_error(TT_UNSUPPORTED, "tt_kv_attention: dtype %lld (TT_F32, TT_BF16, TT_F16)", (long long)a->dtype);
    if (int rc = check_cache("tt_kv_attention", a->cache)) return rc;
    if (a->batch < 0 || a->tokens < 0 || a->table_width < 0 || a->window < 0 || a->sinks < 0)
        return set_error(TT_INVALID, "tt_kv_attention: negative extent");
    if (a->q_heads < 1 || a->q_heads % a->cache.heads)
        return set_error(TT_INVALID, "tt_kv_attention: %lld query heads on %lld cache heads", (long long)a->q_heads,
                         (long long)a->cache.heads);
    if (a->batch == 0 || a->tokens == 0) return TT_OK;
    if (!a->q || !a->out || !a->lengths || (a->table_width > 0 && !a->table))
        return set_error(TT_INVALID, "tt_kv_attention: NULL pointer");
    return TT_OK;
}

}  // namespace
}  // namespace tt

extern "C" size_t tt_kv_attention_workspace_bytes(const tt_kv_attention_args*) { return 0; }

extern "C" int tt_kv_attention(const tt_kv_attention_args* a, void* stream) {
    using namespace tt;
    if (int rc = check_attention(a)) return rc;
    if (a->batch == 0 || a->tokens == 0) return TT_OK;
    AttnParams p;
    p.tokens = a->tokens;
    p.q_heads = a->q_heads;
    p.window = a->window;
    p.sinks = a->sinks;
    p.table_width = a->table_width;
    p.table_stride = a->table_stride;
    for (int i = 0; i < 3; ++i) p.q_stride[i] = a->q_stride[i];
    p.scale = (float)a->scale;
    p.q = a->q;
    p.out = a->out;
    p.table = a->table;
    p.lengths = a->lengths;
    p.counts = a->counts;
    p.c = a->cache;
    p.width = kv_width(a->cache.dim);
    const int64_t rows = a->batch * a->tokens * a->q_heads;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->dtype == TT_F32) return attn_launch<float>(p, rows, st);
    if (a->dtype == TT_BF16) return attn_launch<__bf16>(p, rows, st);
    return attn_launch<_Float16>(p, rows, st);
}
