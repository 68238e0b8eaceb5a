// Attention over a paged cache of 8-bit floats (tt_kv_attention).
//
//   o_r = sum_j softmax_j(scale * q_r . k_j) v_j over the keys j that row r sees
//
// in one pass over the keys with the running maximum and sum of a softmax;
// scores never leave registers, and widened keys and values only, where many
// query rows share them, for LDS.
#include <cmath>
#include <type_traits>

#include "tt_serving.hpp"

namespace tt {

namespace {

struct AttnParams {
    const void* q;
    void* out;
    const int32_t *table, *lengths, *counts;
    const uint8_t *k, *v;
    const float *k_scale, *v_scale;
    float* part;  // partial results: slots of rows * (width + 2) floats
    int64_t q_stride[3], table_stride, pages;
    int batch, tokens, q_heads, heads, share, page, dim, window, sinks, table_width;
    int capacity;    // tokens that the table covers
    int row_blocks;  // blocks of query rows of one cache head
    int groups;      // workgroups that share the key tiles
    int direct;      // each workgroup takes one pair, whole
    FastDiv by_page, by_share;
    float scale;    // magnitude, times log2(e)
    uint32_t flip;  // the sign bits of two 16-bit values where the scale is negative
};

constexpr int kTile = 64;     // keys a wavefront takes at a time
constexpr int kMinTiles = 4;  // fewest tiles worth a workgroup: one per wavefront
// What starting and joining a pair costs, in tiles. 1 to 8 are level within 5%
// at five lengths and batches; 16 takes 90 us for 80 (48 sequences of 4096).
constexpr int kPairCost = 4;

// A value that all lanes of a wavefront share, for scalar registers.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
    return (int64_t)((uint64_t)(uint32_t)uniform((int)x) | (uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32);
}

// Which keys the query rows of one block see: those of [0, end) that are in a
// row's window or among the sinks lie in tiles [0, sink_tiles) and [start, ..).
struct Span {
    int64_t base;              // position of the sequence's first query
    int tokens;                // its queries
    int first_pos, last_pos;   // positions of the block's live rows
    int held;                  // tokens that exist
    int sink_tiles, start, tiles;
    int live;                  // live rows of the block
};

__device__ __forceinline__ Span span_of(const AttnParams& p, int b, int row0, int rows) {
    Span s = {0, 0, 0, -1, 0, 0, 0, 0, 0};
    const int len = p.lengths[b];
    const int n = p.counts ? p.counts[b] : p.tokens;
    s.tokens = n < p.tokens ? n : p.tokens;
    if (s.tokens <= 0 || len <= 0) return s;
    const int64_t all = (int64_t)s.tokens * p.share;
    s.live = all > row0 ? (int)(all - row0 < rows ? all - row0 : rows) : 0;
    if (s.live <= 0) return s;
    s.held = len < p.capacity ? len : p.capacity;
    s.base = (int64_t)len - n;
    const int64_t first = s.base + (int)fdiv(row0, p.by_share), last = s.base + (int)fdiv(row0 + s.live - 1, p.by_share);
    if (last < 0) return s;
    s.first_pos = first < -1 ? -1 : (int)first;
    s.last_pos = (int)last;
    const int end = s.last_pos + 1 < s.held ? s.last_pos + 1 : s.held;
    const int64_t low = p.window > 0 ? (int64_t)s.first_pos - p.window + 1 : 0;
    s.start = low > 0 ? (int)(low / kTile) : 0;
    if (s.start > 0) {
        const int st = p.sinks / kTile + (p.sinks % kTile ? 1 : 0);
        s.sink_tiles = st < s.start ? st : s.start;
    }
    const int last_tile = (end + kTile - 1) / kTile;
    if (last_tile < s.start) s.start = last_tile;
    if (s.sink_tiles > last_tile) s.sink_tiles = last_tile;
    s.tiles = s.sink_tiles + last_tile - s.start;
    return s;
}

// How a dtype's queries and probabilities enter the 16-bit matrix units. Codes
// are exact in either 16-bit type. float32 splits into three bfloat16 parts
// (24 bits); float16 queries are taken as they are, and their probabilities as
// two bfloat16 parts (16 bits), since scaled values may pass float16's range.
// bfloat16 ones are rounded to the 8 bits that their result is held in: two
// parts took 359 us for 270 (2048 tokens on 8192), 52 for 50.5 (48 sequences of
// up to 4096 keys, a token each).
template <typename T>
struct Parts {
    static constexpr int q = 1, p = 1;
    typedef bf16x8 qv;
};
template <>
struct Parts<_Float16> {
    static constexpr int q = 1, p = 2;
    typedef f16x8 qv;
};
template <>
struct Parts<float> {
    static constexpr int q = 3, p = 3;
    typedef bf16x8 qv;
};

template <bool Half>
__device__ __forceinline__ u32x4 widen8(uint32_t lo, uint32_t hi) {
    u32x4 r;
    if constexpr (Half) {
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true));
    } else {
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true));
    }
    return r;
}

__device__ __forceinline__ f32x4 mma_bf16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma_f16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// One wavefront's running state for MT blocks of 16 query rows. With lane l,
// column c = l % 16 is a query row and g = l / 16 a group of four lanes' rows:
//   scores  s[mt][t][r]  key 16 g + 4 t + r of the tile, query row c
//   output  o[mt][d][r]  element 16 d + 4 g + r of query row c
// A tile's keys are dealt to the MFMA rows so that lane group g holds the
// scores of the run of keys 16 g .. 16 g + 15: these are the keys whose values
// the same lane reads as 16 contiguous bytes for the second product, so that
// probabilities pass from one product to the next in their registers, and a
// run lies in one page (pages are multiples of 16), so that a lane needs one
// scale. Keys are read as 16 bytes along d, two products' worth.
//
// What starting and joining a pair compute from the lane and the head size is
// hidden from the compiler (fresh): it would keep the addresses and masks that
// follow, hundreds of registers of them, across the tiles' loop.
__device__ __forceinline__ int fresh(int uniform) {
    asm volatile("" : "+s"(uniform));
    return uniform;
}
__device__ __forceinline__ int fresh_lane(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

template <typename T, int W, int MT>
struct Wave {
    static constexpr int QP = Parts<T>::q, PP = Parts<T>::p;
    static constexpr bool kHalf = std::is_same<T, _Float16>::value;
    u32x4 q[MT][QP][W / 32];
    f32x4 o[MT][W / 16];
    f32x4 l[MT];           // the weights' sum, in every element and lane of a column
    float m[MT];
    uint32_t any[MT];      // not 0 once the row has seen a key
    int end[MT], low[MT];  // this lane's query row sees keys of [0, end) that are >= low or < sinks

    // Rows from row0 on, of which `sp` (the span of them) has the live ones.
    __device__ __forceinline__ void load_q(const AttnParams& p, int b, int kh, int row0, const Span& sp) {
        const int lane = fresh_lane(threadIdx.x & 63), c = lane & 15, h = lane >> 4;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const bool live = mt * 16 + c < sp.live;
            // Rows past the end repeat the first: what they give is not stored.
            const int row = live ? row0 + mt * 16 + c : 0;
            const int t = (int)fdiv(row, p.by_share), g = row - t * p.share;
            const int64_t pos = sp.base + t;
            end[mt] = live && pos >= 0 ? (pos + 1 < sp.held ? (int)pos + 1 : sp.held) : 0;
            const int64_t lo = p.window > 0 ? pos - p.window + 1 : 0;
            low[mt] = lo > 0 ? (int)lo : 0;
            m[mt] = -INFINITY;
            l[mt] = f32x4{0, 0, 0, 0};
            any[mt] = 0;
#pragma unroll
            for (int d = 0; d < W / 16; ++d) o[mt][d] = f32x4{0, 0, 0, 0};
            const T* src = static_cast<const T*>(p.q) + b * p.q_stride[0] + (int64_t)t * p.q_stride[1] +
                           (int64_t)(kh * p.share + g) * p.q_stride[2];
            T x[W / 32][8];
            const int dim = fresh(p.dim);
            if (dim % 8 == 0) {
#pragma unroll
                for (int s = 0; s < W / 32; ++s) {
                    const int d0 = s / 2 * 64 + h * 16 + (s & 1) * 8;
                    __builtin_memcpy(x[s], src + (d0 < dim ? d0 : 0), sizeof x[s]);
                    if (d0 >= dim)
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[s][i] = (T)0.f;
                }
            } else {
#pragma unroll
                for (int s = 0; s < W / 32; ++s)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int d = s / 2 * 64 + h * 16 + (s & 1) * 8 + i;
                        const T v = src[d < dim ? d : 0];
                        x[s][i] = d < dim ? v : (T)0.f;
                    }
            }
#pragma unroll
            for (int s = 0; s < W / 32; ++s) {
                u32x4 parts[QP];
                if constexpr (QP == 1)
                    parts[0] = __builtin_bit_cast(u32x4, x[s]);
                else
                    split8<QP>(x[s], parts);
#pragma unroll
                for (int n = 0; n < QP; ++n) q[mt][n][s] = parts[n] ^ p.flip;
            }
        }
    }
};

// A tile's place in the cache for one lane: the run whose keys it reads as
// rows, and the run whose values (and whose keys' scores) it holds.
struct Runs {
    int k_page, v_page;
};

// First keys of a tile's runs that this lane reads as rows, and whose values it reads.
__device__ __forceinline__ int k_first(int tile) { return tile * kTile + (threadIdx.x >> 2 & 3) * 16; }
__device__ __forceinline__ int v_first(int tile) { return tile * kTile + (threadIdx.x >> 4 & 3) * 16; }

__device__ __forceinline__ Runs find_runs(const AttnParams& p, const int32_t* table, int tile) {
    const int kp = (int)fdiv(k_first(tile), p.by_page), vp = (int)fdiv(v_first(tile), p.by_page);
    return {table[kp < p.table_width ? kp : p.table_width - 1], table[vp < p.table_width ? vp : p.table_width - 1]};
}

// What lies past the sequence's end or in no page is read from page 0 and
// masked; whether the values' run does not.
__device__ __forceinline__ bool settle_runs(const AttnParams& p, Runs& r, int tile, int held) {
    const bool ok = r.v_page >= 0 && r.v_page < p.pages && v_first(tile) < held;
    if (r.k_page < 0 || r.k_page >= p.pages) r.k_page = 0;
    if (!ok) r.v_page = 0;
    return ok;
}

__device__ __forceinline__ const uint8_t* k_run(const AttnParams& p, const Runs& r, int tile, int kh, int W) {
    const int at = k_first(tile), slot = at - (int)fdiv(at, p.by_page) * p.page;
    return p.k + (((int64_t)r.k_page * p.heads + kh) * p.page + slot + (threadIdx.x & 3)) * W + (threadIdx.x >> 4 & 3) * 16;
}

__device__ __forceinline__ const uint8_t* v_run(const AttnParams& p, const Runs& r, int tile, int kh, int W) {
    const int at = v_first(tile), slot = at - (int)fdiv(at, p.by_page) * p.page;
    return p.v + (((int64_t)r.v_page * p.heads + kh) * W + (threadIdx.x & 15)) * p.page + slot;
}

// The scales of the run whose keys' scores a lane holds, as loaded: what is
// made of them is made where they are used, not where that would be a wait for
// them. A value's scale is a power of two, 2^v_exp(): probabilities enter the
// second product times it, and their sums are taken with 2^-v_exp().
struct Scales {
    float k, v;
    bool ok;

    __device__ __forceinline__ float key() const { return ok ? k : 0.f; }
    __device__ __forceinline__ float v_exp() const { return ok ? (float)((int)(__float_as_uint(v) >> 23 & 255) - 127) : 0.f; }
    __device__ __forceinline__ float value() const { return ok ? __uint_as_float(__float_as_uint(v) & 0x7f800000u) : 1.f; }
    // 2^-v_exp() as two bfloat16 values; the low one is that of a float in its upper half.
    __device__ __forceinline__ uint32_t v_inv() const {
        const uint32_t inv = (ok ? 254 - (__float_as_uint(v) >> 23 & 255) : 127u) << 7;
        return inv | inv << 16;
    }
};

__device__ __forceinline__ Scales load_scales(const AttnParams& p, const Runs& r, int kh, bool ok) {
    const int64_t at = (int64_t)r.v_page * p.heads + kh;
    return {p.k_scale[at], p.v_scale[at], ok};
}

template <int W>
struct Tile {
    u32x4 k[4][W / 64], v[W / 16];

    __device__ __forceinline__ void load_k(const uint8_t* src) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int c = 0; c < W / 64; ++c) k[t][c] = *reinterpret_cast<const u32x4*>(src + t * 4 * W + c * 64);
    }
    __device__ __forceinline__ void load_v(const uint8_t* src, int page) {
#pragma unroll
        for (int d = 0; d < W / 16; ++d) {
            v[d] = *reinterpret_cast<const u32x4*>(src);
            src += 16 * page;
        }
    }
};

// Products of one tile's keys with the queries.
template <typename T, int W, int MT>
__device__ __forceinline__ void tile_scores(Wave<T, W, MT>& w, const Tile<W>& x, f32x4 (&s)[MT][4]) {
    typedef Wave<T, W, MT> WV;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int t = 0; t < 4; ++t) s[mt][t] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < W / 64; ++c)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const u32x4 a = widen8<WV::kHalf>(x.k[t][c][2 * u], x.k[t][c][2 * u + 1]);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int n = 0; n < WV::QP; ++n) {
                        if constexpr (WV::kHalf)
                            s[mt][t] = mma_f16(a, w.q[mt][n][2 * c + u], s[mt][t]);
                        else
                            s[mt][t] = mma_bf16(a, w.q[mt][n][2 * c + u], s[mt][t]);
                    }
            }
}

// Bit i: i < n.
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 16 ? 0xffffu : (1u << n) - 1; }

// Four bits as the low bits of four bytes.
__device__ __forceinline__ uint32_t bits_to_bytes(uint32_t m) { return (m & 15u) * 0x00204081u & 0x01010101u; }

// Bytes that are NaN codes, as 1.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t v) { return ((v & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u; }

// A tile that some row does not see whole: bit i of mask[mt] says whether this
// lane's row sees key i of its run. Values of keys that no row of the wavefront
// sees may be anything, so zeros are put in their place (`keep`: the bytes that
// stay). NaN among the others belongs only to the rows that see it: it is
// zeroed as well, and those rows' output set to NaN through a product of its
// places with `seen` (1.0 where the row sees the key).
template <int MT>
struct Edge {
    uint32_t keep[4];
    u32x4 seen[MT][2];

    __device__ __forceinline__ explicit Edge(const uint32_t (&mask)[MT]) {
        uint32_t some = mask[0];
#pragma unroll
        for (int mt = 1; mt < MT; ++mt) some |= mask[mt];
        some |= __builtin_amdgcn_mov_dpp(some, 0x128, 0xf, 0xf, true);  // row_ror: over the 16 columns
        some |= __builtin_amdgcn_mov_dpp(some, 0x124, 0xf, 0xf, true);
        some |= __builtin_amdgcn_mov_dpp(some, 0x122, 0xf, 0xf, true);
        some |= __builtin_amdgcn_mov_dpp(some, 0x121, 0xf, 0xf, true);
#pragma unroll
        for (int i = 0; i < 4; ++i) keep[i] = bits_to_bytes(some >> 4 * i) * 0xffu;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                seen[mt][i / 4][i % 4] = (mask[mt] >> 2 * i & 1 ? 0x3f80u : 0u) | (mask[mt] >> 2 * i & 2 ? 0x3f800000u : 0u);
    }
    // Clears the codes v of one block of 16 elements and tells of NaN among the rest.
    __device__ __forceinline__ uint32_t clear(u32x4& v) const {
        uint32_t nan = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] &= keep[i];
            nan |= nan_bytes(v[i]);
        }
        return nan;
    }
    // Takes NaN out of cleared codes, o[mt] being the block's output.
    __device__ __forceinline__ u32x4 settle_nan(u32x4 v, f32x4 (&o)[MT]) const {
        u32x4 flag;
        uint32_t nan = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t at = nan_bytes(v[i]);
            flag[i] = at * 0x38u;  // the code of 1.0
            v[i] &= ~(at * 0xffu);
            nan |= at;
        }
        if (__any(nan != 0)) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                f32x4 hit = {0, 0, 0, 0};
#pragma unroll
                for (int h = 0; h < 2; ++h) hit = mma_bf16(widen8<false>(flag[2 * h], flag[2 * h + 1]), seen[mt][h], hit);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (hit[r] > 0.f) o[mt][r] = NAN;
            }
        }
        return v;
    }
};

// Which keys of its run a lane's rows see of a tile, and scores of the others set to -inf.
template <typename T, int W, int MT>
__device__ __forceinline__ void mask_scores(const AttnParams& p, Wave<T, W, MT>& w, bool ok, f32x4 (&s)[MT][4], int tile,
                                            uint32_t (&mask)[MT]) {
    const int key0 = tile * kTile + (threadIdx.x >> 4 & 3) * 16;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        mask[mt] = ok ? bits_below(w.end[mt] - key0) & (~bits_below(w.low[mt] - key0) | bits_below(p.sinks - key0)) : 0u;
        w.any[mt] |= mask[mt];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t on = (uint32_t)((int)(mask[mt] << (31 - i)) >> 31);
            s[mt][i / 4][i % 4] = __uint_as_float((__float_as_uint(s[mt][i / 4][i % 4]) & on) | (0xff800000u & ~on));
        }
    }
}

// The weights of one tile's keys, of products s (-inf where masked), as the
// operands of the second product, and their sum and maximum in the running
// state. What is summed are the weights as that product takes them: rounding
// then moves a result in proportion to how far values lie from it, not to
// their size.
template <typename T, int W, int MT>
__device__ __forceinline__ void tile_weights(const AttnParams& p, Wave<T, W, MT>& w, const Scales& sc, f32x4 (&s)[MT][4],
                                             u32x4 (&prob)[MT][Wave<T, W, MT>::PP][2]) {
    typedef Wave<T, W, MT> WV;
    // Not zero, so that a masked score stays -inf whatever the scale.
    const float c = fmaxf(sc.key() * p.scale, 1e-30f);
    const uint32_t inv = sc.v_inv();
    const u32x4 one = {inv, inv, inv, inv};
    // A value's scale enters as a term of the exponent, which then has up to 7
    // bits fewer behind the point (2^-18 of a weight at a scale of 2^-64), below
    // what the parts of 16-bit types keep; float32 weights are multiplied by it.
    constexpr bool kApart = sizeof(T) == 4;
    const float v_exp = kApart ? 0.f : sc.v_exp(), v_scale = kApart ? sc.value() : 1.f;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        float top = s[mt][0][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[mt][i / 4][i % 4]);
        top *= c;
        // The maximum is moved only where some score passes it by over 8 (its
        // weight would be over 256): until then weights and sums keep it.
        const float m_old = w.m[mt];
        if (__any(top > m_old + 8.f)) {
            const float m_new = fmaxf(m_old, column_max(top));
            const float keep = m_new == -INFINITY ? 1.f : exp2f(m_old - m_new);
            w.m[mt] = m_new;
            w.l[mt] *= keep;
#pragma unroll
            for (int d = 0; d < W / 16; ++d) w.o[mt][d] *= keep;
        }
        const float shift = v_exp - (w.m[mt] == -INFINITY ? 0.f : w.m[mt]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mt][2 * h + i / 4][i & 3], c, shift));
            if constexpr (kApart) {
#pragma unroll
                for (int i = 0; i < 8; ++i) e[i] *= v_scale;
            }
            u32x4 parts[WV::PP];
            split8<WV::PP>(e, parts);
#pragma unroll
            for (int n = 0; n < WV::PP; ++n) {
                prob[mt][n][h] = parts[n];
                w.l[mt] = mma_bf16(one, parts[n], w.l[mt]);
            }
        }
    }
}

__device__ __forceinline__ int tile_at(const Span& sp, int i) { return i < sp.sink_tiles ? i : sp.start + i - sp.sink_tiles; }

// Keys [low, end) are seen by every live row of a span, as are those below the sinks' end.
struct Sure {
    int low, end;

    __device__ __forceinline__ Sure(const AttnParams& p, const Span& sp) {
        end = sp.first_pos + 1 < sp.held ? sp.first_pos + 1 : sp.held;
        const int64_t lo = p.window > 0 ? (int64_t)sp.last_pos - p.window + 1 : 0;
        low = lo > 0 ? (int)lo : 0;
    }
    __device__ __forceinline__ bool sees(const AttnParams& p, int tile) const {
        const int key = tile * kTile;
        return key + kTile <= end && (key >= low || key + kTile <= p.sinks);
    }
};

// Folds tiles first, first + step, ... below last of the span into the wave's
// state; `r` is where the first of them lies.
template <typename T, int W, int MT>
__device__ __forceinline__ void walk(const AttnParams& p, Wave<T, W, MT>& w, const Span& sp, int b, int kh, Runs r,
                                     int first, int last, int step) {
    typedef Wave<T, W, MT> WV;
    if (first >= last) return;
    const int32_t* table = p.table + b * p.table_stride;
    const Sure sure(p, sp);
    Tile<W> x;
    // Loads return in order, so what is needed first is asked for first: the
    // pages of the tile after next, this tile's values, the next one's keys.
    int tile = tile_at(sp, first), next = tile_at(sp, first + step < last ? first + step : first);
    Scales sc = load_scales(p, r, kh, settle_runs(p, r, tile, sp.held));
    x.load_k(k_run(p, r, tile, kh, W));
    Runs rn = find_runs(p, table, next);
    for (int i = first; i < last; i += step) {
        const int after = i + 2 * step < last ? tile_at(sp, i + 2 * step) : next;
        const Runs ra = find_runs(p, table, after);
        x.load_v(v_run(p, r, tile, kh, W), p.page);
        __builtin_amdgcn_sched_barrier(0);  // in flight while the scores are formed
        f32x4 s[MT][4];
        tile_scores<T, W, MT>(w, x, s);
        const Scales now = sc;
        // (After the last tile it is loaded again: with the same loads in flight
        // on every path, the wait for the values need not be one for the keys.)
        r = rn;
        const bool ok = settle_runs(p, r, next, sp.held);
        sc = load_scales(p, r, kh, ok);
        x.load_k(k_run(p, r, next, kh, W));
        rn = ra;
        __builtin_amdgcn_sched_barrier(0);  // in flight while the tile is folded
        const bool full = sure.sees(p, tile) && __all(now.ok);
        if (full) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) w.any[mt] = 1;
        } else {
            uint32_t mask[MT];
            mask_scores<T, W, MT>(p, w, now.ok, s, tile, mask);
            const Edge<MT> edge(mask);
            uint32_t nan = 0;
#pragma unroll
            for (int d = 0; d < W / 16; ++d) nan |= edge.clear(x.v[d]);
            if (__any(nan != 0)) {
#pragma unroll
                for (int d = 0; d < W / 16; ++d) {
                    f32x4 o[MT];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) o[mt] = w.o[mt][d];
                    x.v[d] = edge.settle_nan(x.v[d], o);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) w.o[mt][d] = o[mt];
                }
            }
        }
        u32x4 prob[MT][WV::PP][2];
        tile_weights<T, W, MT>(p, w, now, s, prob);
#pragma unroll
        for (int d = 0; d < W / 16; ++d)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const u32x4 a = widen8<false>(x.v[d][2 * h], x.v[d][2 * h + 1]);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int n = 0; n < WV::PP; ++n) w.o[mt][d] = mma_bf16(a, prob[mt][n][h], w.o[mt][d]);
            }
        tile = next;
        next = after;
    }
}

template <typename T>
__device__ __forceinline__ void store4(T* dst, const float* v, int count) {
    if (count >= 4) {
        T x[4] = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
        __builtin_memcpy(dst, x, sizeof x);
    } else {
        for (int i = 0; i < count; ++i) dst[i] = (T)v[i];
    }
}

// Address of query row `row` of (b, kh) in the contiguous output.
template <typename T>
__device__ __forceinline__ T* out_row(const AttnParams& p, int b, int kh, int row) {
    const int t = (int)fdiv(row, p.by_share), g = row - t * p.share;
    return static_cast<T*>(p.out) + (((int64_t)b * p.tokens + t) * p.q_heads + kh * p.share + g) * p.dim;
}

template <typename T, int W>
__device__ __forceinline__ void zero_rows(const AttnParams& p, int b, int kh, int row0, int row1) {
    const int rows = p.tokens * p.share;
    if (row1 > rows) row1 = rows;
    for (int i = fresh_lane(threadIdx.x); i < (row1 - row0) * W; i += 256) {
        const int d = i % W;
        if (d < p.dim) out_row<T>(p, b, kh, row0 + i / W)[d] = (T)0.f;
    }
}

// The four wavefronts' states of the same 16 query rows, joined; to the output
// or to a slot of partial results.
template <typename T, int W>
__device__ __forceinline__ void join_waves(const AttnParams& p, Wave<T, W, 1>& w, const Span& sp, int b, int kh, int row0,
                                           float* slot) {
    __shared__ float sm[4][16], sl[4][16];
    __shared__ float so[4][16][68];
    const int tid = fresh_lane(threadIdx.x), dim = fresh(p.dim);
    const int lane = tid & 63, wave = uniform(tid >> 6), c = lane & 15, g = lane >> 4;
    const float l = w.l[0][0];
    const bool any = column_sum(w.any[0] ? 1.f : 0.f) > 0.f;
    if (g == 0) {
        sm[wave][c] = w.m[0];
        sl[wave][c] = any ? l : -1.f;
    }
    __syncthreads();
    float m = -INFINITY, sum = 0.f;
    bool some = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, sm[i][c]);
    const float shift = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool has = sl[i][c] != -1.f;
        if (has) sum += sl[i][c] * exp2f(sm[i][c] - shift);
        some |= has;
    }
    const float mine = any ? exp2f(w.m[0] - shift) * (slot ? 1.f : 1.f / sum) : 0.f;
    if (slot && tid < 16 && c < sp.live) {
        slot[16 * W + c] = m;
        slot[16 * W + 16 + c] = some ? sum : -1.f;
    }
    const int oc = tid >> 4, od = (tid & 15) * 4;
#pragma unroll
    for (int d0 = 0; d0 < W / 64; ++d0) {
        if (d0) __syncthreads();
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            f32x4 v = any ? w.o[0][d0 * 4 + d] * mine : f32x4{0, 0, 0, 0};
            *reinterpret_cast<f32x4*>(&so[wave][c][d * 16 + g * 4]) = v;
        }
        __syncthreads();
        f32x4 v = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) v += *reinterpret_cast<const f32x4*>(&so[i][oc][od]);
        if (oc < sp.live) {
            if (slot) {
                *reinterpret_cast<f32x4*>(slot + oc * W + d0 * 64 + od) = v;
            } else {
                float x[4] = {v[0], v[1], v[2], v[3]};
                const int d = d0 * 64 + od;
                if (d < dim) store4<T>(out_row<T>(p, b, kh, row0 + oc) + d, x, dim - d);
            }
        }
    }
    __syncthreads();
}

// The work of a sequence's pairs, in tiles, and of all sequences.
__device__ __forceinline__ int64_t weight_of(const AttnParams& p, int b) {
    const int tiles = span_of(p, b, 0, 16).tiles;
    return tiles > 0 ? (int64_t)(tiles + kPairCost) * p.heads : 0;
}

struct Weights {
    int64_t total, before;  // of all sequences, and of those before a given one
};

// By one wavefront.
__device__ __forceinline__ Weights all_weights(const AttnParams& p, int limit) {
    Weights w = {0, 0};
    for (int b = threadIdx.x & 63; b < p.batch; b += 64) {
        const int64_t v = weight_of(p, b);
        w.total += v;
        if (b < limit) w.before += v;
    }
    for (int off = 32; off > 0; off >>= 1) {
        w.total += __shfl_xor(w.total, off, 64);
        w.before += __shfl_xor(w.before, off, 64);
    }
    return {uniform(w.total), uniform(w.before)};
}

__device__ __forceinline__ int64_t share_of(const AttnParams& p, int64_t total) {
    const int64_t per = (total + p.groups - 1) / p.groups;
    return per < kMinTiles + kPairCost ? kMinTiles + kPairCost : per;
}

// Wavefronts a SIMD is to hold: two where the state of one fits half its registers.
template <typename T, int W, int MT>
constexpr int kWavesPerSimd = Parts<T>::q * MT * W > 256 || W > 128 ? 1 : 2;

// Few query rows (at most 16 a cache head): the four wavefronts of a workgroup
// take every fourth tile of the same keys. The key tiles of all (sequence,
// head) pairs form one list, in which each pair also takes the room of what
// starting it costs; the workgroups share it evenly whatever the sequences'
// lengths, and a pair cut by a workgroup's end leaves partial results. Or, for
// short tables, each takes a pair whole (cut_of). Bound by the codes' bytes: two
// sequences of 131071 tokens (8 heads of 128, 534 MB) take 106 us, 5.0 TB/s where
// a large copy has 5.2; 48 of 1 to 4096, a workgroup a pair, 50 us, 4.0 TB/s, the
// longest pairs being left at the end (all of 4096: 5.2 TB/s at head size 256);
// one of 200 tokens 7 us, the launch and a chain of waits (length, page, keys,
// values). 256 pairs of 18 tiles (windows) leave one wavefront a SIMD, which
// waits on memory 57% of its time.
template <typename T, int W>
__global__ __launch_bounds__(256, (kWavesPerSimd<T, W, 1>)) void kv_attention_few_kernel(AttnParams p) {
    const int wave = uniform((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    Wave<T, W, 1> w;
    // This workgroup's places [pos, stop) of the list, and sequence b, whose first pair is at `at`.
    int64_t pos, stop, at = 0;
    int b = 0;
    Span sp;
    Runs r;
    if (p.direct) {
        b = blockIdx.x / p.heads;
        // Where a wavefront's first tile lies is looked up beside the lengths
        // (without a window: which tile it is follows from nothing else).
        if (p.capacity > 0) r = find_runs(p, p.table + b * p.table_stride, wave);
        sp = span_of(p, b, 0, 16);
        const int kh = blockIdx.x - b * p.heads;
        zero_rows<T, W>(p, b, kh, sp.tiles > 0 ? sp.live : 0, 16);
        pos = (int64_t)kh * (sp.tiles + kPairCost);
        stop = sp.tiles > 0 ? pos + sp.tiles + kPairCost : pos;
    } else {
        const int64_t total = all_weights(p, p.batch).total, per = share_of(p, total);
        pos = blockIdx.x * per;
        stop = pos + per < total ? pos + per : total;
        // Rows that see nothing: their zeros, dealt out over the workgroups.
        for (int i = blockIdx.x; i < p.batch; i += gridDim.x) {
            const Span z = span_of(p, i, 0, 16);
            if (z.tiles == 0 || z.live < 16)
                for (int kh = 0; kh < p.heads; ++kh) zero_rows<T, W>(p, i, kh, z.tiles == 0 ? 0 : z.live, 16);
        }
        if (pos >= stop) return;
        for (int b0 = 0;; b0 += 64) {
            const int64_t mine = b0 + lane < p.batch ? weight_of(p, b0 + lane) : 0;
            int64_t upto = mine;
            for (int off = 1; off < 64; off <<= 1) {
                const int64_t v = __shfl_up(upto, off, 64);
                upto += lane >= off ? v : 0;
            }
            const uint64_t past = __ballot(at + upto > pos);
            if (past) {
                const int f = __builtin_ctzll(past);
                b = b0 + f;
                at += uniform((int64_t)__shfl(upto - mine, f, 64));
                break;
            }
            at += uniform((int64_t)__shfl(upto, 63, 64));
        }
    }
    while (pos < stop) {
        if (!p.direct) sp = span_of(p, b, 0, 16);
        const int64_t pair_weight = sp.tiles + kPairCost, size = sp.tiles > 0 ? pair_weight * p.heads : 0;
        if (pos >= at + size) {
            at += size;
            ++b;
            continue;
        }
        const int kh = (int)((pos - at) / pair_weight);
        const int64_t pair = at + kh * pair_weight + kPairCost, end = stop < pair + sp.tiles ? stop : pair + sp.tiles;
        const int first = pos > pair ? (int)(pos - pair) : 0, last = end > pair ? (int)(end - pair) : 0;
        pos = end > pos ? end : stop;
        if (first >= last) continue;
        if (!p.direct || p.window > 0) r = find_runs(p, p.table + b * p.table_stride, tile_at(sp, first + wave));
        w.load_q(p, b, kh, 0, sp);
        walk<T, W, 1>(p, w, sp, b, kh, r, first + wave, last, 4);
        // A pair is cut at most at this workgroup's ends: in its first or its last tiles.
        const bool whole = first == 0 && last == sp.tiles;
        float* slot = whole ? nullptr : p.part + ((int64_t)blockIdx.x * 2 + (first == 0 ? 1 : 0)) * (16 * (W + 2));
        join_waves<T, W>(p, w, sp, b, kh, 0, slot);
    }
}

// One query row of `parts` partial results by one wavefront: slot 0 is `first`
// and slot i > 0 `rest` + i * stride; a slot holds its rows' sums of W elements,
// and the row's maximum and weight at m_at and l_at (weight -1: no key seen).
// kDeep slots are in flight.
template <typename T, int W, int kDeep>
__device__ __forceinline__ void join_row(const float* first, const float* rest, int64_t stride, int parts, int row, int m_at,
                                         int l_at, int dim, T* out) {
    const int lane = threadIdx.x & 63;
    auto slot = [&](int i) { return i ? rest + i * stride : first; };
    float x[kDeep][W / 64];
    auto load = [&](int i) {
#pragma unroll
        for (int u = 0; u < kDeep; ++u) {
            const float* s = slot(i + u < parts ? i + u : parts - 1) + row * W + lane;
#pragma unroll
            for (int d = 0; d < W / 64; ++d) x[u][d] = s[d * 64];
        }
    };
    // The first elements, maxima and weights are asked for together: which
    // memory they come from is a longer way than what is done with them.
    const float* own = slot(lane < parts ? lane : parts - 1);
    float m = own[m_at];
    const float m_own = m, l_own = own[l_at];
    load(0);
    __builtin_amdgcn_sched_barrier(0);
    for (int i = lane + 64; i < parts; i += 64) m = fmaxf(m, slot(i)[m_at]);
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    const float shift = m == -INFINITY ? 0.f : m;
    float sum = 0.f, o[W / 64] = {};
    bool some = false;
    for (int i0 = 0; i0 < parts; i0 += 64) {
        float f = 0.f;
        if (i0 + lane < parts) {
            const float* s = slot(i0 + lane);
            const float l = i0 ? s[l_at] : l_own;
            if (l != -1.f) {
                f = exp2f((i0 ? s[m_at] : m_own) - shift);
                sum += l * f;
                some = true;
            }
        }
        const int n = parts - i0 < 64 ? parts - i0 : 64;
        for (int i = 0; i < n; i += kDeep) {
            if (i0 + i > 0) load(i0 + i);
#pragma unroll
            for (int u = 0; u < kDeep; ++u) {
                if (i + u >= n) break;
                const float g = __shfl(f, i + u, 64);
#pragma unroll
                for (int d = 0; d < W / 64; ++d) o[d] += g * x[u][d];
            }
        }
    }
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    some = __any(some);
#pragma unroll
    for (int d = 0; d < W / 64; ++d)
        if (d * 64 + lane < dim) out[d * 64 + lane] = (T)(some ? o[d] / sum : 0.f);
}

// Joins the partial results of the pairs that were cut: one wavefront a query
// row. A launch and two waits on memory (lengths, partial results): 5 us where
// nothing is cut, 8 for 32 partial results of each of 16 pairs.
template <typename T, int W>
__global__ __launch_bounds__(256) void kv_attention_few_join_kernel(AttnParams p) {
    constexpr int64_t kSlot = 16 * (W + 2);
    const int b = blockIdx.x / p.heads, kh = blockIdx.x - b * p.heads;
    const Span sp = span_of(p, b, 0, 16);
    const Weights w = all_weights(p, b);
    if (sp.tiles == 0) return;
    const int64_t per = share_of(p, w.total);
    const int64_t pair = w.before + kh * (int64_t)(sp.tiles + kPairCost) + kPairCost;
    const int64_t g0 = pair / per, g1 = (pair + sp.tiles - 1) / per;
    if (g0 == g1) return;
    const float* base = p.part + g0 * 2 * kSlot;
    for (int row = uniform((int)threadIdx.x >> 6); row < sp.live; row += 4)
        join_row<T, W, 32>(base + kSlot, base, 2 * kSlot, (int)(g1 - g0 + 1), row, 16 * W + row, 16 * W + 16 + row, p.dim,
                       out_row<T>(p, b, kh, row));
}

// Many query rows: each of NW wavefronts takes MT blocks of 16 rows, and all of
// them walk the same keys, whose codes the workgroup widens once and puts into
// LDS as the operands of the products, tile by tile in two buffers: what widens
// a tile, loads it and reads it is shared by 16 MT NW rows. With `groups` > 1
// the keys of a row block are cut into that many ranges, joined afterwards. 2048
// tokens on 8192 (32 heads of 128, 240 GFLOP): 268 us, 0.90 PFLOP/s of the 1.22
// that a large product reaches. Bound by issue: the products take the matrix
// units 44% of a wavefront's time, exponentials, widening and addresses the
// vector units 41%, and with two wavefronts a SIMD the two overlap in part only.
// float16 takes 354 us and float32 571, head sizes of 64, 192 and 256 193, 417
// and 500 (bfloat16): rows of more than 128 codes and float32 have no room for
// two blocks of rows a wavefront.
template <typename T, int W, int MT, int NW>
__global__ __launch_bounds__(64 * NW, (NW == 8 ? 2 : 1)) void kv_attention_many_kernel(AttnParams p) {
    typedef Wave<T, W, MT> WV;
    constexpr int kRows = 16 * MT * NW;
    constexpr int kKeys = W / 16, kLoads = 2 * kKeys, kMine = kLoads / NW;  // 16-byte pieces a lane: of keys, of a tile, a wavefront's
    static_assert(kLoads % NW == 0, "pieces divide evenly");
    __shared__ u32x4 lds[2][2 * kLoads][64];
    __shared__ int nan_values[3];  // whether tile n's values, if some row does not see them all, hold NaN: at n % 3
    const int wave = uniform((int)threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    int id = blockIdx.x;
    const int part = id % p.groups;
    id /= p.groups;
    const int kh = id % p.heads;
    id /= p.heads;
    // The last row blocks of a sequence see the most keys: they go first.
    const int b = id % p.batch, rb = p.row_blocks - 1 - id / p.batch;
    const int row0 = rb * kRows, mine = row0 + wave * 16 * MT;
    const Span all = span_of(p, b, row0, kRows);
    const int per = all.tiles > 0 ? (all.tiles + p.groups - 1) / p.groups : 1;
    const int first = part * per, last = first + per < all.tiles ? first + per : all.tiles;
    if (part > 0 && first >= last) return;
    WV w;
    const Span sp = span_of(p, b, mine, 16 * MT);
    w.load_q(p, b, kh, mine, sp);
    if (first < last) {
        const int32_t* table = p.table + b * p.table_stride;
        const Sure sure(p, all);
        const int end = all.last_pos + 1 < all.held ? all.last_pos + 1 : all.held;  // no row sees further
        u32x4 raw[kMine];
        Scales sc;
        // Piece n of a tile: of its keys (row block n % 4, elements 64 (n / 4) ..) or, from kKeys on, of its values.
        auto load = [&](const Runs& r, int tile, bool ok) {
            sc = load_scales(p, r, kh, ok);
            const uint8_t *k = k_run(p, r, tile, kh, W), *v = v_run(p, r, tile, kh, W);
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const int n = wave + i * NW;
                const uint8_t* src = n < kKeys ? k + n % 4 * 4 * W + n / 4 * 64 : v + (int64_t)(n - kKeys) * 16 * p.page;
                raw[i] = *reinterpret_cast<const u32x4*>(src);
            }
        };
        auto stage = [&](int n, int tile, bool ok) {
            const int buffer = n & 1;
            uint32_t nan = 0;
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const int piece = wave + i * NW;
                u32x4 x = raw[i];
                if (piece < kKeys) {
                    const int at = piece % 4 * (W / 32) + piece / 4 * 2;
                    lds[buffer][at][lane] = widen8<WV::kHalf>(x[0], x[1]);
                    lds[buffer][at + 1][lane] = widen8<WV::kHalf>(x[2], x[3]);
                } else {
                    if (!sure.sees(p, tile) || !ok) {
                        const uint32_t live = ok ? bits_below(end - tile * kTile - g * 16) : 0u;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            x[j] &= bits_to_bytes(live >> 4 * j) * 0xffu;
                            const uint32_t at = nan_bytes(x[j]);
                            nan |= at;
                            x[j] &= ~(at * 0xffu);
                        }
                    }
                    const int at = kLoads + (piece - kKeys) * 2;
                    lds[buffer][at][lane] = widen8<false>(x[0], x[1]);
                    lds[buffer][at + 1][lane] = widen8<false>(x[2], x[3]);
                }
            }
            if (nan) nan_values[n % 3] = 1;
        };
        if (threadIdx.x < 3) nan_values[threadIdx.x] = 0;
        __syncthreads();
        const int tiles = last - first;
        auto tile_of = [&](int n) { return tile_at(all, first + (n < tiles ? n : tiles - 1)); };
        int tile = tile_of(0);
        Runs r = find_runs(p, table, tile);
        const bool ok = settle_runs(p, r, tile, all.held);
        load(r, tile, ok);
        stage(0, tile, ok);
        Scales now = sc;
        Runs at = r;
        r = find_runs(p, table, tile_of(1));
        f32x4 s[MT][4];
        __syncthreads();
        auto scores = [&](const u32x4(*keys)[64]) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int t = 0; t < 4; ++t) s[mt][t] = f32x4{0, 0, 0, 0};
            u32x4 a[2][4];
#pragma unroll
            for (int t = 0; t < 4; ++t) a[0][t] = keys[t * (W / 32)][lane];
#pragma unroll
            for (int e = 0; e < W / 32; ++e) {
                if (e + 1 < W / 32) {
#pragma unroll
                    for (int t = 0; t < 4; ++t) a[(e + 1) & 1][t] = keys[t * (W / 32) + e + 1][lane];
                }
                __builtin_amdgcn_sched_barrier(0);  // read a step ahead
#pragma unroll
                for (int n = 0; n < WV::QP; ++n)
#pragma unroll
                    for (int t = 0; t < 4; ++t)
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            if constexpr (WV::kHalf)
                                s[mt][t] = mma_f16(a[e & 1][t], w.q[mt][n][e], s[mt][t]);
                            else
                                s[mt][t] = mma_bf16(a[e & 1][t], w.q[mt][n][e], s[mt][t]);
                        }
            }
        };
        // Between two barriers, tile n of the walk is worked on in buffer n % 2 and
        // tile n + 1 loaded, then staged in the other.
        for (int n = 0; n < tiles; ++n) {
            const bool more = n + 1 < tiles;
            const int next = tile_of(n + 1);
            const bool fits = settle_runs(p, r, next, all.held);
            const Runs after = r;
            r = find_runs(p, table, tile_of(n + 2));
            load(after, next, fits);
            __builtin_amdgcn_sched_barrier(0);  // in flight while this tile is worked on
            scores(lds[n & 1]);
            const bool full = sure.sees(p, tile) && __all(now.ok);
            uint32_t mask[MT];
            if (full) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) w.any[mt] = 1;
            } else {
                mask_scores<T, W, MT>(p, w, now.ok, s, tile, mask);
            }
            u32x4 prob[MT][WV::PP][2];
            tile_weights<T, W, MT>(p, w, now, s, prob);
            if (!full && nan_values[n % 3]) {
                // Values staged without their NaN, which not every row
                // sees: it is given to those that do.
                const Edge<MT> edge(mask);
                const uint8_t* v = v_run(p, at, tile, kh, W);
#pragma unroll
                for (int d = 0; d < W / 16; ++d) {
                    f32x4 o[MT];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) o[mt] = w.o[mt][d];
                    u32x4 x = *reinterpret_cast<const u32x4*>(v + (int64_t)d * 16 * p.page);
                    edge.clear(x);
                    edge.settle_nan(x, o);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) w.o[mt][d] = o[mt];
                    __builtin_amdgcn_sched_barrier(0);  // one at a time: registers matter more
                }
            }
            const u32x4(*values)[64] = lds[n & 1] + kLoads;
            u32x4 a[2][2] = {{values[0][lane], values[1][lane]}};
#pragma unroll
            for (int d = 0; d < W / 16; ++d) {
                if (d + 1 < W / 16) {
                    a[(d + 1) & 1][0] = values[d * 2 + 2][lane];
                    a[(d + 1) & 1][1] = values[d * 2 + 3][lane];
                }
                __builtin_amdgcn_sched_barrier(0);  // read a block ahead
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int i = 0; i < WV::PP; ++i) w.o[mt][d] = mma_bf16(a[d & 1][h], prob[mt][i][h], w.o[mt][d]);
            }
            // Marks of NaN: tile n's is read here, n + 1's set, n + 2's cleared.
            if (threadIdx.x == 0) nan_values[(n + 2) % 3] = 0;
            if (more) stage(n + 1, next, fits);
            now = sc;
            at = after;
            tile = next;
            __syncthreads();
        }
    }
    float* slot = p.groups > 1 && per < all.tiles
                      ? p.part + ((((int64_t)b * p.row_blocks + rb) * p.heads + kh) * p.groups + part) * (kRows * (W + 2))
                      : nullptr;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int row = wave * 16 * MT + mt * 16 + c;
        const float l = w.l[mt][0];
        const bool any = column_sum(w.any[mt] ? 1.f : 0.f) > 0.f;
        if (row0 + row >= p.tokens * p.share) continue;
        const bool dead = row >= all.live || !any;
        if (slot) {
            if (g == 0) {
                slot[kRows * W + row] = w.m[mt];
                slot[kRows * W + kRows + row] = dead ? -1.f : l;
            }
#pragma unroll
            for (int d = 0; d < W / 16; ++d) *reinterpret_cast<f32x4*>(slot + row * W + d * 16 + g * 4) = w.o[mt][d];
        } else {
            const int dim = fresh(p.dim);
            T* out = out_row<T>(p, b, kh, row0 + row);
            const float f = 1.f / l;
#pragma unroll
            for (int d = 0; d < W / 16; ++d) {
                const int d0 = d * 16 + g * 4;
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = dead ? 0.f : w.o[mt][d][i] * f;
                if (d0 < dim) store4<T>(out + d0, x, dim - d0);
            }
        }
    }
}

template <typename T, int W, int kRows>
__global__ __launch_bounds__(256) void kv_attention_many_join_kernel(AttnParams p) {
    int id = blockIdx.x;
    const int chunk = id % (kRows / 4);
    id /= kRows / 4;
    const int kh = id % p.heads;
    id /= p.heads;
    const int rb = id % p.row_blocks, b = id / p.row_blocks;
    const int row0 = rb * kRows, r = chunk * 4 + uniform((int)threadIdx.x >> 6);
    const Span all = span_of(p, b, row0, kRows);
    if (row0 + r >= p.tokens * p.share || all.tiles <= 0) return;
    const int per = (all.tiles + p.groups - 1) / p.groups;
    if (per >= all.tiles) return;
    constexpr int64_t kSlot = kRows * (W + 2);
    const float* base = p.part + (((int64_t)b * p.row_blocks + rb) * p.heads + kh) * p.groups * kSlot;
    join_row<T, W, 8>(base, base, kSlot, (all.tiles + per - 1) / per, r, kRows * W + r, kRows * W + kRows + r, p.dim,
                   out_row<T>(p, b, kh, row0 + r));
}

// Workgroups of many rows: blocks of 16 rows a wavefront, wavefronts, and the
// us that a tile takes with one workgroup on a compute unit and, where two fit,
// with two (bfloat16, head size 128). Eight wavefronts of two blocks widen a
// tile for the most rows (2048 tokens on 8192: 268 us, of one block 340, four
// of one 396); smaller blocks waste less where rows are few or the causal edge
// is steep (128 tokens on 1024: 27, 22, 20; 2048 on 2048: 80, 64, 76).
struct Shape {
    int mt, waves;
    double alone, both;
};
constexpr Shape kShapes[] = {{1, 4, 1.27, 1.85}, {1, 8, 1.47, 1.47}, {2, 8, 2.15, 2.15}};

// What a call is expected to take (us), its keys cut into g ranges. Joining
// them is a second launch that reads what the first one wrote: 5 us, 0.36 a MB
// and 0.45 a thousand rows. It pays where blocks leave compute units idle (one
// block a head, 8192 keys: 278 us whole, 34 in 32 ranges), not where keys are
// few for their rows (eight times 128 tokens on 1024: 32 us whole, 56 halved).
// `width` and `kind` say what 2048 tokens on 8192 take at head sizes 64 to 256
// within 10% for bfloat16 (256: 14%) and 16% for float16, against the same shape
// at 128 in bfloat16; float32 of more than 128 codes a row, which has one shape,
// takes a third longer. Keys
// are those that the table covers: sequences that are shorter have ranges of
// few tiles (512 tokens on 512 through a table of 4096 keys or more 33 us, of
// 512 17; 128 on 1024 29 for 19).
double many_cost(const tt_kv_attention_args* a, const Shape& s, int64_t W, int64_t tiles, int64_t blocks, int64_t g,
                 int64_t slots) {
    const double width = (W + 64) / 192.0, kind = a->dtype == TT_F32 ? 1.6 : a->dtype == TT_F16 ? 1.3 : 1.0;
    const double per = (double)((tiles + g - 1) / g), cap = (double)a->table_width * a->cache.page;
    // Of a prompt's own keys its rows see half.
    const double seen = a->window > 0 || cap <= 0 ? 1 : 1 - 0.5 * (a->tokens < cap ? a->tokens : cap) / cap;
    const int64_t n = blocks * g, rounds = (n + slots - 1) / slots;
    const double start = 2;  // tiles' worth, of every workgroup
    const double longest = (per + start) * s.alone, all = (per * seen + start) * rounds * (n <= 256 ? s.alone : s.both);
    const double rows = 16.0 * s.mt * s.waves * blocks;
    const double join = g > 1 ? 5 + 0.36e-6 * rows * g * (W + 2) * 4 + 0.45e-3 * rows : 0;
    return (longest > all ? longest : all) * width * kind + join;
}

// How a call is cut, from what the host knows of it.
struct Cut {
    bool few, direct;
    int mt, waves, row_blocks, groups;
    int64_t grid, join, slots, slot_floats;  // workgroups, and those that join partial results
};

Cut cut_of(const tt_kv_attention_args* a) {
    Cut c = {};
    const int64_t share = a->q_heads / a->cache.heads, rows = a->tokens * share, W = kv_width(a->cache.dim);
    const int64_t cap = a->table_width * a->cache.page;
    int64_t keys = cap;  // the most a row block may have to walk
    if (a->window > 0 && a->window < cap && a->sinks < cap) {
        const int64_t w = a->window + a->sinks + a->tokens + 2 * kTile;
        keys = w < cap ? w : cap;
    }
    const int64_t tiles = (keys + kTile - 1) / kTile;
    const int64_t pairs = a->batch * a->cache.heads;
    c.few = rows <= 16;
    if (c.few) {
        c.mt = 1;
        c.row_blocks = 1;
        // A workgroup a pair needs no second launch to join (about 5 us), but
        // lets its longest pair decide. us direct / shared, one token of 8 heads
        // of 128: 8 pairs of 1024 keys 10.8 / 14.4, of 2048 15.4 / 14.1; 64 pairs
        // of 2048 17.6 / 18.6, of 4096 30.2 / 24.6; 256 pairs of 4096 43.7 / 52.8
        // (of 1 to 4096 33.6 / 36.0), 512 of 4096 100.7 / 106.3 (57.2 / 61.9);
        // past what is resident at once, 1024 pairs of 4096 241 / 198, but 2048
        // of 1500 134 / 170. The table's width is all the host knows of the
        // lengths: beyond 64 tiles one long sequence among short ones would
        // hold up its few workgroups. (That bound is this worry's; what was
        // measured does not cross there.) Short sequences in a table past the
        // bound pay for the join: 200 keys 12 us, in a table of 1024 keys 7.
        const int most = pairs < 64 ? 16 : pairs < 256 || pairs > 512 ? 32 : 64;
        c.direct = tiles <= most;
        c.groups = 512;  // two a compute unit; 256 and 1024 were 8% slower at some length each, level at others
        c.grid = c.direct ? pairs : c.groups;
        c.join = c.direct ? 0 : pairs;
        c.slots = c.direct ? 0 : 2 * c.groups;
        c.slot_floats = 16 * (W + 2);
    } else {
        c.mt = c.waves = 0;
        double best = 0;
        for (const Shape& s : kShapes) {
            if ((s.mt == 2 && (W > 128 || a->dtype == TT_F32)) || (s.waves == 8 && W > 128 && a->dtype == TT_F32)) continue;
            const int64_t block = 16 * s.mt * s.waves, blocks = pairs * ((rows + block - 1) / block);
            if (c.waves && rows <= block / 2) continue;
            const int64_t slots = s.waves == 4 && W <= 128 ? 512 : 256, fit = slots / blocks;
            for (int64_t g = 1;; g = 2 * g < fit ? 2 * g : fit) {
                const double cost = many_cost(a, s, W, tiles, blocks, g, slots);
                if (!c.waves || cost < best) {
                    best = cost;
                    c.mt = s.mt;
                    c.waves = s.waves;
                    c.groups = (int)g;
                    c.row_blocks = (int)(blocks / pairs);
                }
                if (g >= fit || 2 * g > tiles) break;
            }
        }
        const int64_t block = 16 * c.mt * c.waves, blocks = pairs * c.row_blocks;
        c.grid = blocks * c.groups;
        c.join = c.groups > 1 ? blocks * 4 * c.mt * c.waves : 0;
        c.slots = c.groups > 1 ? blocks * c.groups : 0;
        c.slot_floats = block * (W + 2);
    }
    return c;
}

template <typename T, int W, int MT, int NW>
int attn_many(const AttnParams& p, const Cut& c, hipStream_t st) {
    kv_attention_many_kernel<T, W, MT, NW><<<(uint32_t)c.grid, 64 * NW, 0, st>>>(p);
    if (c.join) kv_attention_many_join_kernel<T, W, 16 * MT * NW><<<(uint32_t)c.join, 256, 0, st>>>(p);
    return check_launch("tt_kv_attention");
}

template <typename T, int W>
int attn_launch(const AttnParams& p, const Cut& c, hipStream_t st) {
    if (c.few) {
        kv_attention_few_kernel<T, W><<<(uint32_t)c.grid, 256, 0, st>>>(p);
        if (c.join) kv_attention_few_join_kernel<T, W><<<(uint32_t)c.join, 256, 0, st>>>(p);
        return check_launch("tt_kv_attention");
    }
    if (c.waves == 4) return attn_many<T, W, 1, 4>(p, c, st);
    if constexpr (sizeof(T) == 2 && W <= 128)
        if (c.mt == 2) return attn_many<T, W, 2, 8>(p, c, st);
    if constexpr (sizeof(T) == 2 || W <= 128) return attn_many<T, W, 1, 8>(p, c, st);
    return set_error(TT_HIP_ERROR, "tt_kv_attention: no kernel");
}

template <typename T>
int attn_typed(AttnParams& p, const Cut& c, hipStream_t st) {
    switch (kv_width(p.dim)) {
        case 64:
            return attn_launch<T, 64>(p, c, st);
        case 128:
            return attn_launch<T, 128>(p, c, st);
        case 192:
            return attn_launch<T, 192>(p, c, st);
        default:
            return attn_launch<T, 256>(p, c, st);
    }
}

int check_attention(const tt_kv_attention_args* a) {
    if (!a) return set_error(TT_INVALID, "tt_kv_attention: NULL arguments");
    if (!serving_dtype(a->dtype))
        return set_error(TT_UNSUPPORTED, "tt_kv_attention: dtype %lld (TT_F32, TT_BF16, TT_F16)", (long long)a->dtype);
    if (int rc = check_cache("tt_kv_attention", a->cache)) return rc;
    if (a->batch < 0 || a->tokens < 0 || a->table_width < 0 || a->window < 0 || a->sinks < 0)
        return set_error(TT_INVALID, "tt_kv_attention: negative extent");
    if (!(std::fabs(a->scale) < 1e38)) return set_error(TT_INVALID, "tt_kv_attention: scale %g", a->scale);
    if (a->q_heads < 1 || a->q_heads % a->cache.heads)
        return set_error(TT_INVALID, "tt_kv_attention: %lld query heads on %lld cache heads", (long long)a->q_heads,
                         (long long)a->cache.heads);
    if (a->batch == 0 || a->tokens == 0) return TT_OK;
    if (!a->q || !a->out || !a->lengths || (a->table_width > 0 && !a->table))
        return set_error(TT_INVALID, "tt_kv_attention: NULL pointer");
    constexpr int64_t kMost = int64_t(1) << 30;
    if (a->batch >= kMost || a->tokens >= kMost || a->q_heads >= kMost || a->batch * a->cache.heads >= kMost ||
        a->tokens * a->q_heads >= kMost || a->cache.pages >= kMost || a->table_width > kMost / a->cache.page)
        return set_error(TT_UNSUPPORTED, "tt_kv_attention: extents of 2^30 or more");
    return TT_OK;
}

}  // namespace
}  // namespace tt

extern "C" size_t tt_kv_attention_workspace_bytes(const tt_kv_attention_args* a) {
    using namespace tt;
    if (check_attention(a) != TT_OK || a->batch == 0 || a->tokens == 0) return 0;
    const Cut c = cut_of(a);
    return (size_t)(c.slots * c.slot_floats * 4);
}

extern "C" int tt_kv_attention(const tt_kv_attention_args* a, void* stream) {
    using namespace tt;
    if (int rc = check_attention(a)) return rc;
    if (a->batch == 0 || a->tokens == 0) return TT_OK;
    const Cut c = cut_of(a);
    const int64_t most = c.waves > 4 ? kMaxGrid / 2 : kMaxGrid;  // of eight wavefronts: half as many
    if (c.grid > most || c.join > kMaxGrid)
        return set_error(TT_UNSUPPORTED, "tt_kv_attention: %lld workgroups", (long long)(c.grid > c.join ? c.grid : c.join));
    const int64_t need = c.slots * c.slot_floats * 4;
    if (need > 0 && (!a->workspace || a->workspace_bytes < need || (uintptr_t)a->workspace % 16))
        return set_error(TT_INVALID, "tt_kv_attention: workspace of %lld bytes, need %lld", (long long)a->workspace_bytes,
                         (long long)need);
    AttnParams p;
    p.q = a->q;
    p.out = a->out;
    p.table = a->table;
    p.lengths = a->lengths;
    p.counts = a->counts;
    p.k = static_cast<const uint8_t*>(a->cache.k);
    p.v = static_cast<const uint8_t*>(a->cache.v);
    p.k_scale = a->cache.k_scale;
    p.v_scale = a->cache.v_scale;
    p.part = static_cast<float*>(a->workspace);
    for (int i = 0; i < 3; ++i) p.q_stride[i] = a->q_stride[i];
    p.table_stride = a->table_stride;
    p.pages = a->cache.pages;
    p.batch = (int)a->batch;
    p.tokens = (int)a->tokens;
    p.q_heads = (int)a->q_heads;
    p.heads = (int)a->cache.heads;
    p.share = p.q_heads / p.heads;
    p.page = (int)a->cache.page;
    p.dim = (int)a->cache.dim;
    constexpr int64_t kInt = 0x7fffffff;
    p.window = (int)(a->window < kInt ? a->window : kInt);
    p.sinks = (int)(a->sinks < kInt ? a->sinks : kInt);
    p.capacity = a->cache.pages > 0 ? (int)(a->table_width * a->cache.page) : 0;
    p.table_width = (int)a->table_width;
    p.row_blocks = c.row_blocks;
    p.groups = c.groups;
    p.direct = c.direct;
    p.by_page = make_fastdiv((uint32_t)p.page);
    p.by_share = make_fastdiv((uint32_t)p.share);
    p.scale = (float)((a->scale < 0 ? -a->scale : a->scale) * 1.4426950408889634074);
    p.flip = a->scale < 0 ? 0x80008000u : 0u;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->dtype == TT_F32) return attn_typed<float>(p, c, st);
    if (a->dtype == TT_BF16) return attn_typed<__bf16>(p, c, st);
    return attn_typed<_Float16>(p, c, st);
}
