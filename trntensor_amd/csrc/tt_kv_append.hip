// Appending keys and values to a paged cache of 8-bit floats, with the
// position rotation of keys and queries on the way.
#include "tt_serving.hpp"

namespace tt {

namespace {

struct AppendParams {
    int64_t batch, tokens, q_heads, rot, interleaved, table_width, table_stride;
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

// What one workgroup of the cache part appends to: the new tokens [lo, hi) of
// one block (page and head), keys or values.
struct Block {
    bool is_v;
    int lo, hi;         // slots of the page
    int64_t first;      // position of the page's first slot
    const void* x;      // row of slot 0 (its head), which need not exist
    int64_t row_stride;
    uint8_t* codes;
    float* scale;
};

// (Extents and lengths fit 32 bits: a 64-bit division is a hundred instructions.)
template <typename T>
__device__ __forceinline__ bool find_block(const AppendParams& p, uint32_t w, Block& k) {
    const uint32_t H = (uint32_t)p.c.heads, P = (uint32_t)p.c.page, blocks = (uint32_t)p.blocks;
    k.is_v = w & 1;
    w >>= 1;
    const uint32_t pair = w / H, h = w - pair * H, b = pair / blocks, j = pair - b * blocks;
    const int64_t len = p.lengths[b];
    int64_t n = p.counts ? p.counts[b] : p.tokens;
    n = n > p.tokens ? p.tokens : n;
    if (len < 0) return false;
    const int64_t end = len + n < p.table_width * P ? len + n : p.table_width * P;
    const int64_t block = (uint32_t)len / P + j;
    k.first = block * P;
    k.lo = (int)((len > k.first ? len : k.first) - k.first);
    const int64_t hi = (end < k.first + P ? end : k.first + P) - k.first;
    if (k.lo >= hi) return false;
    k.hi = (int)hi;
    const int64_t page = p.table[b * p.table_stride + block];
    if (page < 0 || page >= p.c.pages) return false;
    const int64_t* stride = k.is_v ? p.v_stride : p.k_stride;
    k.x = static_cast<const T*>(k.is_v ? p.v : p.k) + b * stride[0] + h * stride[2] + (k.first - len) * stride[1];
    k.row_stride = stride[1];
    k.codes = static_cast<uint8_t*>(k.is_v ? p.c.v : p.c.k) + (page * H + h) * p.width * P;
    k.scale = (k.is_v ? p.c.v_scale : p.c.k_scale) + page * H + h;
    return true;
}

// The largest magnitude as bits, which order as magnitudes do; anything from
// 0x7f800000 on says that an infinity or NaN is among them.
constexpr uint32_t kNotFinite = 0x7f800000u;

__device__ __forceinline__ void take_max(uint32_t& top, float x) {
    const uint32_t a = __float_as_uint(x) & 0x7fffffffu;
    top = a > top ? a : top;
}

__device__ __forceinline__ void take_finite_max(uint32_t& top, float x) {
    const uint32_t a = __float_as_uint(x) & 0x7fffffffu;
    if (a < kNotFinite) top = a > top ? a : top;
}

// Over the workgroup.
__device__ __forceinline__ uint32_t top_of_all(uint32_t top) {
    __shared__ uint32_t part[4];
    for (int off = 32; off > 0; off >>= 1) {
        const uint32_t o = __shfl_xor(top, off, 64);
        top = o > top ? o : top;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x / 64] = top;
    __syncthreads();
    const uint32_t a = part[0] > part[1] ? part[0] : part[1], b = part[2] > part[3] ? part[2] : part[3];
    return a > b ? a : b;
}

// The block's new scale: its new values' (the largest finite magnitude's), or
// its old one if that is larger and the block holds earlier tokens.
__device__ __forceinline__ float new_scale(uint32_t top, float old) {
    return fmaxf(power_of_two(scale_exponent(__uint_as_float(top))), old);
}

// Four values as codes. Finite ones are within the format's range at their
// block's scale; with others about (`wild`) each is saturated.
__device__ __forceinline__ uint32_t codes_of(const float* x, float inv, bool wild) {
    const float a = x[0] * inv, b = x[1] * inv, c = x[2] * inv, d = x[3] * inv;
    if (wild) return fp8_pair(a, b) | fp8_pair(c, d) << 16;
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}

// Four codes at another scale.
__device__ __forceinline__ uint32_t rescaled(uint32_t c, float f) {
    const uint32_t lo = fp8_pair(__builtin_amdgcn_cvt_f32_fp8(c, 0) * f, __builtin_amdgcn_cvt_f32_fp8(c, 1) * f);
    const uint32_t hi = fp8_pair(__builtin_amdgcn_cvt_f32_fp8(c, 2) * f, __builtin_amdgcn_cvt_f32_fp8(c, 3) * f);
    return lo | hi << 16;
}

// Element by element, for head sizes and rotations that are no multiples of
// the pieces below.
template <typename T>
__global__ __launch_bounds__(256) void kv_append_any_kernel(AppendParams p) {
    const int64_t P = p.c.page, W = p.width;
    if (blockIdx.x >= p.kv_groups) {
        const int64_t w = blockIdx.x - p.kv_groups, b = w / p.tokens, t = w % p.tokens;
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
    Block k;
    if (!find_block<T>(p, blockIdx.x, k)) return;
    const T* x = static_cast<const T*>(k.x);
    auto value = [&](int64_t t, int d) -> float {
        if (d >= p.c.dim) return 0.f;
        return k.is_v ? to_f32(x[t * k.row_stride + d]) : rotated<T>(p, x + t * k.row_stride, k.first + t, d);
    };
    auto place = [&](int64_t t, int64_t d) { return k.is_v ? d * P + t : t * W + d; };
    const float old = k.lo > 0 ? *k.scale : 0.f;
    uint32_t top = 0;
    for (int64_t i = k.lo * W + threadIdx.x; i < k.hi * W; i += 256) take_finite_max(top, value(i / W, (int)(i % W)));
    const float scale = new_scale(top_of_all(top), old), inv = 1.f / scale;
    if (k.lo > 0 && scale > old) {
        for (int64_t i = threadIdx.x; i < k.lo * W; i += 256) {
            uint8_t* c = k.codes + place(i / W, i % W);
            *c = (uint8_t)fp8_pair(fp8_value(*c) * (old * inv), 0.f);
        }
    }
    for (int64_t i = k.lo * W + threadIdx.x; i < k.hi * W; i += 256) {
        const int64_t t = i / W, d = i % W;
        k.codes[place(t, d)] = (uint8_t)fp8_pair(value(t, (int)d) * inv, 0.f);
    }
    if (threadIdx.x == 0) *k.scale = scale;
}

template <typename T>
__device__ __forceinline__ void load8(const T* src, float* x) {
    T v[8];
    __builtin_memcpy(v, src, sizeof v);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(v[i]);
}

// Eight elements as they lie in memory.
template <typename T>
struct Eight {
    u32x4 raw[sizeof(T) / 2];

    __device__ __forceinline__ Eight() {}
    __device__ __forceinline__ explicit Eight(const float* v) {
        T t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = (T)v[i];
        __builtin_memcpy(raw, t, sizeof raw);
    }
    __device__ __forceinline__ void load(const T* src) { __builtin_memcpy(raw, src, sizeof raw); }
    __device__ __forceinline__ void store(T* dst) const { __builtin_memcpy(dst, raw, sizeof raw); }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(raw[i / 4][i % 4]);
        if constexpr (sizeof(T) == 2) {
            const uint16_t h = (uint16_t)(raw[0][i / 2] >> 16 * (i & 1));
            return to_f32(__builtin_bit_cast(T, h));
        }
    }
};

// The two pieces of eight elements that one thread takes of a row: for the
// rotated part a piece and the one it is paired with (the same distance into
// the other half, or its neighbour), after that neighbours.
struct Pieces {
    int a, b;   // first elements
    int turn;   // first of their cos and sin, or -1
};

__device__ __forceinline__ Pieces pieces_of(const AppendParams& p, int i, bool rotate) {
    const int rot = rotate ? (int)p.rot : 0;
    if (16 * i >= rot) return {16 * i, 16 * i + 8, -1};
    if (p.interleaved) return {16 * i, 16 * i + 8, 8 * i};
    return {8 * i, 8 * i + rot / 2, 8 * i};
}

// Rotates the pieces a and b by eight angles; each product and sum is rounded.
__device__ __forceinline__ void turn_pieces(const float* c, const float* s, bool interleaved, float* a, float* b) {
#pragma clang fp contract(off)
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a0 = a[2 * i], a1 = a[2 * i + 1], b0 = b[2 * i], b1 = b[2 * i + 1];
            const float p0 = a0 * c[i], p1 = a1 * s[i], p2 = a1 * c[i], p3 = a0 * s[i];
            const float r0 = b0 * c[4 + i], r1 = b1 * s[4 + i], r2 = b1 * c[4 + i], r3 = b0 * s[4 + i];
            a[2 * i] = p0 - p1;
            a[2 * i + 1] = p2 + p3;
            b[2 * i] = r0 - r1;
            b[2 * i + 1] = r2 + r3;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float p0 = a[i] * c[i], p1 = b[i] * s[i], p2 = b[i] * c[i], p3 = a[i] * s[i];
            a[i] = p0 - p1;
            b[i] = p2 + p3;
        }
    }
}

// The queries of one token, rotated, by a wavefront (see kv_append_kernel).
template <typename T, int W>
__device__ __forceinline__ void rotate_token(const AppendParams& p, int64_t row) {
    constexpr int kRow = W / 16;  // lanes a head
    const int tid = threadIdx.x, D = (int)p.c.dim;
    const uint32_t tokens = (uint32_t)p.tokens;
    const int64_t b = (uint32_t)row / tokens, t = (uint32_t)row - (uint32_t)b * tokens;
    if (b >= p.batch) return;
    const int64_t n = p.counts ? p.counts[b] : p.tokens, pos = (int64_t)p.lengths[b] + t;
    const bool live = t < n && pos >= 0 && pos < p.table_width * p.c.page;
    const T* q = static_cast<const T*>(p.q) + b * p.q_stride[0] + t * p.q_stride[1];
    T* out = static_cast<T*>(p.q_out) + row * p.q_heads * D;
    constexpr int kLanes = 64 / kRow * kRow;  // lanes at work: whole rows
    const int lane = tid & 63;
    if (lane >= kLanes) return;
    const Pieces at = pieces_of(p, lane % kRow, true);
    float c[8], s[8];
    if (live && at.turn >= 0) {
        __builtin_memcpy(c, p.cos + pos * (p.rot / 2) + at.turn, sizeof c);
        __builtin_memcpy(s, p.sin + pos * (p.rot / 2) + at.turn, sizeof s);
    }
    constexpr int kHeads = 64 / kRow;
    constexpr int kDeep = 2;  // heads of a lane in flight: more take more registers (four: 97 us for 95)
    for (int h0 = lane / kRow; h0 < p.q_heads; h0 += kDeep * kHeads) {
        Eight<T> x[kDeep][2];
#pragma unroll
        for (int u = 0; u < kDeep; ++u) {
            const int h = h0 + u * kHeads;
            const T* src = q + h * p.q_stride[2];
            if (live && h < p.q_heads) {
                if (at.a < D) x[u][0].load(src + at.a);
                if (at.b < D) x[u][1].load(src + at.b);
            }
        }
#pragma unroll
        for (int u = 0; u < kDeep; ++u) {
            const int h = h0 + u * kHeads;
            if (h >= p.q_heads) break;
            float v[2][8];
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i / 8][i % 8] = live ? x[u][i / 8].get(i % 8) : 0.f;
            if (live && at.turn >= 0) turn_pieces(c, s, p.interleaved, v[0], v[1]);
            if (at.a < D) Eight<T>(v[0]).store(out + (int64_t)h * D + at.a);
            if (at.b < D) Eight<T>(v[1]).store(out + (int64_t)h * D + at.b);
        }
    }
}

template <typename T, int W>
__global__ __launch_bounds__(256) void rotate_queries_kernel(AppendParams p) {
    rotate_token<T, W>(p, (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6));
}

// Bytes-bound: keys, values and queries are read once, codes and rotated
// queries written once.
//   keys     a thread takes 16 elements of a token at a time and keeps them in
//            registers between the block's maximum and its codes
//   values   a thread takes two neighbouring elements of the 16 tokens of a
//            run, whose codes lie together in the cache
//   queries  a wavefront takes a token; a lane's elements are in the same
//            place of every head, so that it reads its angles once
// Four prompts of 4096 tokens (8 heads of 128, 32 query heads, 377 MB) take 95
// us, 4.0 TB/s where a large copy has 5.2: the queries wait on memory 87% of
// their time, keys and values (32 us alone, 3.2 TB/s) 69%, between a load, a
// maximum over the workgroup and a store. One token of eight sequences takes 5
// us, a launch and the waits for length, page, scale and values one after the
// other. Head sizes are multiples of 8 here and rotated parts of 16; others
// (head size 100: 332 us for the same prompts) go element by element.
template <typename T, int W, bool Queries>
__global__ __launch_bounds__(256, (Queries ? 2 : 4)) void kv_append_kernel(AppendParams p) {
    constexpr int kRow = W / 16;  // threads a row
    const int tid = threadIdx.x, D = (int)p.c.dim;
    if (Queries && blockIdx.x >= p.kv_groups) {
        rotate_token<T, W>(p, (int64_t)(blockIdx.x - p.kv_groups) * 4 + (tid >> 6));
        return;
    }
    Block k;
    if (!find_block<T>(p, blockIdx.x, k)) return;
    const T* x = static_cast<const T*>(k.x);
    const float old = k.lo > 0 ? *k.scale : 0.f;
    uint32_t top = 0;
    if (!k.is_v) {
        // keys
        constexpr int kHold = 2;  // rows of threads held in registers
        const Pieces at = pieces_of(p, tid % kRow, p.cos != nullptr);
        auto load = [&](int t, float* v) {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = 0.f;
            const T* src = x + t * k.row_stride;
            if (at.a < D) load8(src + at.a, v);
            if (at.b < D) load8(src + at.b, v + 8);
            if (at.turn >= 0) {
                float c[8], s[8];
                __builtin_memcpy(c, p.cos + (k.first + t) * (p.rot / 2) + at.turn, sizeof c);
                __builtin_memcpy(s, p.sin + (k.first + t) * (p.rot / 2) + at.turn, sizeof s);
                turn_pieces(c, s, p.interleaved, v, v + 8);
            }
        };
        constexpr int kStep = 256 / kRow;  // rows a pass
        const int t0 = tid < kStep * kRow ? k.lo + tid / kRow : k.hi;
        float held[kHold][16];
#pragma unroll
        for (int u = 0; u < kHold; ++u)
            if (t0 + u * kStep < k.hi) load(t0 + u * kStep, held[u]);
#pragma unroll
        for (int u = 0; u < kHold; ++u)
            if (t0 + u * kStep < k.hi)
#pragma unroll
                for (int i = 0; i < 16; ++i) take_max(top, held[u][i]);
        for (int t = t0 + kHold * kStep; t < k.hi; t += kStep) {
            float v[16];
            load(t, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) take_max(top, v[i]);
        }
        top = top_of_all(top);
        const bool wild = top >= kNotFinite;
        if (wild) {
            uint32_t finite = 0;
            for (int t = t0; t < k.hi; t += kStep) {
                float v[16];
                load(t, v);
#pragma unroll
                for (int i = 0; i < 16; ++i) take_finite_max(finite, v[i]);
            }
            top = top_of_all(finite);
        }
        const float scale = new_scale(top, old), inv = 1.f / scale;
        auto store = [&](int t, const float* v) {
            u32x2 a = {codes_of(v, inv, wild), codes_of(v + 4, inv, wild)};
            u32x2 b = {codes_of(v + 8, inv, wild), codes_of(v + 12, inv, wild)};
            *reinterpret_cast<u32x2*>(k.codes + (int64_t)t * W + at.a) = a;
            *reinterpret_cast<u32x2*>(k.codes + (int64_t)t * W + at.b) = b;
        };
#pragma unroll
        for (int u = 0; u < kHold; ++u)
            if (t0 + u * kStep < k.hi) store(t0 + u * kStep, held[u]);
        for (int t = t0 + kHold * kStep; t < k.hi; t += kStep) {
            float v[16];
            load(t, v);
            store(t, v);
        }
        if (k.lo > 0 && scale > old) {
            for (int64_t i = tid; i < (int64_t)k.lo * W / 4; i += 256) {
                uint32_t* c = reinterpret_cast<uint32_t*>(k.codes) + i;
                *c = rescaled(*c, old * inv);
            }
        }
        if (tid == 0) *k.scale = scale;
        return;
    }
    // values
    const int run0 = k.lo / 16, runs = (k.hi + 15) / 16 - run0, P = (int)p.c.page;
    struct Run {
        T two[16][2];
    };
    // Two elements of a run's 16 tokens, zeros in other slots.
    auto load = [&](int unit, Run& v) {
        const int t = (run0 + unit / (W / 2)) * 16, d = unit % (W / 2) * 2;
        const T* src = x + t * k.row_stride + d;
        if (d < D && t >= k.lo && t + 16 <= k.hi) {
#pragma unroll
            for (int i = 0; i < 16; ++i) __builtin_memcpy(v.two[i], src + i * k.row_stride, sizeof v.two[i]);
            return;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            v.two[i][0] = v.two[i][1] = (T)0.f;
            if (d < D && t + i >= k.lo && t + i < k.hi) __builtin_memcpy(v.two[i], src + i * k.row_stride, sizeof v.two[i]);
        }
    };
    auto each = [&](const Run& v, auto take, uint32_t& most) {
#pragma unroll
        for (int i = 0; i < 32; ++i) take(most, to_f32(v.two[i / 2][i & 1]));
    };
    const int units = runs * (W / 2);
    Run held;
    if (tid < units) {
        load(tid, held);
        each(held, take_max, top);
    }
    for (int u = tid + 256; u < units; u += 256) {
        Run v;
        load(u, v);
        each(v, take_max, top);
    }
    top = top_of_all(top);
    const bool wild = top >= kNotFinite;
    if (wild) {
        uint32_t finite = 0;
        for (int u = tid; u < units; u += 256) {
            Run v;
            load(u, v);
            each(v, take_finite_max, finite);
        }
        top = top_of_all(finite);
    }
    const float scale = new_scale(top, old), inv = 1.f / scale;
    const bool grown = k.lo > 0 && scale > old;
    for (int u = tid; u < units; u += 256) {
        if (u != tid) load(u, held);
        const int t = (run0 + u / (W / 2)) * 16, d = u % (W / 2) * 2;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            u32x4* dst = reinterpret_cast<u32x4*>(k.codes + (int64_t)(d + e) * P + t);
            u32x4 c;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = to_f32(held.two[4 * i + j][e]);
                c[i] = codes_of(v, inv, wild);
            }
            if (t < k.lo || t + 16 > k.hi) {
                // a run that holds other tokens: earlier ones, or slots not yet taken
                const u32x4 was = *dst;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int slot = t + 4 * i;
                    auto below = [&](int n) { return n <= slot ? 0u : n >= slot + 4 ? ~0u : (1u << 8 * (n - slot)) - 1; };
                    const uint32_t earlier = below(k.lo), taken = below(k.hi);
                    const uint32_t again = grown ? rescaled(was[i], old * inv) : was[i];
                    c[i] = (again & earlier) | (c[i] & taken & ~earlier) | (was[i] & ~taken);
                }
            }
            *dst = c;
        }
    }
    if (grown) {
        // runs of earlier tokens only
        for (int64_t u = tid; u < (int64_t)run0 * W; u += 256) {
            u32x4* dst = reinterpret_cast<u32x4*>(k.codes + u / run0 * P + u % run0 * 16);
            u32x4 c = *dst;
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] = rescaled(c[i], old * inv);
            *dst = c;
        }
    }
    if (tid == 0) *k.scale = scale;
}

// A few workgroups are one launch. Many are two, so that neither kind holds the
// other's registers: four prompts of 4096 tokens took 108 us as one launch and
// 95 as two, one token of eight sequences 4.9 us as one.
constexpr int64_t kOneLaunch = 2048;

template <typename T, int W>
int append_width(const AppendParams& p, int64_t rows, hipStream_t st) {
    const int64_t groups = (rows + 3) / 4;
    if (p.kv_groups + groups <= kOneLaunch) {
        kv_append_kernel<T, W, true><<<(uint32_t)(p.kv_groups + groups), 256, 0, st>>>(p);
    } else {
        kv_append_kernel<T, W, false><<<(uint32_t)p.kv_groups, 256, 0, st>>>(p);
        if (groups) rotate_queries_kernel<T, W><<<(uint32_t)groups, 256, 0, st>>>(p);
    }
    return check_launch("tt_kv_append");
}

template <typename T>
int append_launch(const AppendParams& p, bool queries, hipStream_t st) {
    const int64_t rows = queries ? p.batch * p.tokens : 0;
    const bool any = p.c.dim % 8 != 0 || p.rot % 16 != 0;
    // (kv_groups is within a launch's limit; four rows of queries are a workgroup, those of a launch of their own.)
    const int64_t grid = any ? p.kv_groups + rows : (rows + 3) / 4;
    if (grid > kMaxGrid) return set_error(TT_UNSUPPORTED, "tt_kv_append: %lld workgroups", (long long)grid);
    if (any) {
        kv_append_any_kernel<T><<<(uint32_t)(p.kv_groups + rows), 256, 0, st>>>(p);
        return check_launch("tt_kv_append");
    }
    switch (p.width) {
        case 64:
            return append_width<T, 64>(p, rows, st);
        case 128:
            return append_width<T, 128>(p, rows, st);
        case 192:
            return append_width<T, 192>(p, rows, st);
        default:
            return append_width<T, 256>(p, rows, st);
    }
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
    p.batch = a->batch;
    p.tokens = a->tokens;
    p.q_heads = a->q_heads;
    p.rot = a->cos ? a->rot : 0;
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
    if (a->batch > kMaxGrid || a->tokens > kMaxGrid || a->cache.heads > kMaxGrid / a->batch ||
        p.blocks > kMaxGrid / 2 / (a->batch * a->cache.heads))
        return set_error(TT_UNSUPPORTED, "tt_kv_append: %lld sequences of %lld tokens", (long long)a->batch,
                         (long long)a->tokens);
    p.kv_groups = 2 * a->batch * a->cache.heads * p.blocks;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->dtype == TT_F32) return append_launch<float>(p, a->q != nullptr, st);
    if (a->dtype == TT_BF16) return append_launch<__bf16>(p, a->q != nullptr, st);
    return append_launch<_Float16>(p, a->q != nullptr, st);
}
