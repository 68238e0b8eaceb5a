// Products of many rows in 8 bits with 8-bit weights, and the gated block on
// two of them: workgroup tiles whose operands are copied global -> LDS by
// direct loads.
//
// A workgroup has WM x WN wavefronts of MB x NB blocks of 16 x 16. A stage is one
// block of 128 columns: rows of x as eight 16-byte pieces, piece p of row r at
// position p ^ (r / 2 % 8) so that 16 lanes' reads cover 256 bytes, and weight
// tiles as they are packed. Two stages are held; a step multiplies one of them:
//   the rows' blocks two at a time, the next two being read from LDS meanwhile;
//   before the last two, all reads of the stage are done and the next stage has
//   arrived: one barrier, behind which this stage's slot is filled again (two
//   steps ahead) and the next stage's weights and first rows are read while the
//   last two blocks are multiplied.
// The rows' scales come along in fours of blocks, 4 bytes a row.
#include <type_traits>

#include "tt_fp8_block.hpp"

namespace tt {

namespace {

__device__ __forceinline__ unsigned lds_address(const void* p) {
    return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// Direct loads, 16 and 4 bytes a lane, to LDS address `to` (uniform) + 16 or 4 *
// lane, from base (uniform) + offset. They are assembly so that the compiler
// does not take them for writes that every LDS read has to wait for; the
// kernel's own waits and barriers order them. Nothing else here uses M0.
__device__ __forceinline__ void copy16(unsigned to, const uint8_t* base, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(to), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void copy4(unsigned to, const uint8_t* base, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, %2" : : "s"(to), "v"(offset), "s"(base) : "memory", "m0");
}

// s_waitcnt immediates: vmcnt in bits 3:0 and 15:14, expcnt 6:4 (7: no wait), lgkmcnt 11:8.
constexpr int wait_vm(int n) { return (n & 15) | (n >> 4) << 14 | 0xf70; }
constexpr int kWaitAll = 0x70;  // vmcnt(0) lgkmcnt(0)

__device__ __forceinline__ const uint8_t* uniform_ptr(const uint8_t* p) {
    const uint64_t v = (uint64_t)(uintptr_t)p;
    return (const uint8_t*)(uintptr_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)v) |
                                       (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32);
}

struct Codes {};  // the result's type where it is rows in 8 bits

template <typename T, bool E8, bool GATED, int WM, int WN, int MB, int NB>
__global__ __launch_bounds__(64 * WM * WN, 2) void fp8_tiles_kernel(Fp8Params p, int tiles_m, int tiles_n) {
    constexpr bool CODES = std::is_same<T, Codes>::value, EXACT = std::is_same<T, float>::value;
    constexpr int NW = WM * WN, BM = WM * MB * 16;
    constexpr int NT = WN * NB;                          // weight tiles of 16 rows a stage
    constexpr int BN = GATED ? NT * 8 : NT * 16;         // columns of the result
    constexpr int XB = BM * 128, WB = NT * 2048;         // bytes a stage
    constexpr int XI = XB / 1024 / NW, WI = WB / 1024 / NW;  // direct loads a wavefront a stage
    constexpr int SI = (BM + 63) / 64;                   // direct loads of a four of scales, one a wavefront
    constexpr int PH = MB / 2;
    static_assert(XI * 1024 * NW == XB && WI * 1024 * NW == WB && SI <= NW && MB % 2 == 0, "tile");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * XB + 2 * WB + 2 * BM * 4];
    const unsigned lds0 = lds_address(lds), ldsw = lds0 + 2 * XB, ldss = ldsw + 2 * WB;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const int wm = wave / WN, wn = wave % WN;

    // Each XCD walks a contiguous range of tiles, four tiles of rows at a time.
    const int total = tiles_m * tiles_n;
    const int id = (int)xcd_remap(blockIdx.x, total);
    constexpr int kGroup = 4;
    const int grp = id / (kGroup * tiles_n), rest = id - grp * kGroup * tiles_n;
    const int high = tiles_m - grp * kGroup < kGroup ? tiles_m - grp * kGroup : kGroup;
    const int m0 = (grp * kGroup + rest % high) * BM, n0 = rest / high * BN;

    // What this lane's direct loads read: rows past the end repeat the last one,
    // weight tiles past the end the last one, and what they give is not stored.
    const int64_t pitch = (int64_t)p.blocks * 128;
    const uint8_t* x_base = p.x + m0 * pitch;
    uint32_t x_off[XI];
#pragma unroll
    for (int i = 0; i < XI; ++i) {
        const int r = (wave * XI + i) * 8 + (lane >> 3);
        const int row = m0 + r < p.M ? r : p.M - 1 - m0;
        x_off[i] = (uint32_t)(row * pitch) + (((lane & 7) ^ (r >> 1 & 7)) * 16);
    }
    const int last_tile = (p.N + 15) / 16 - 1;
    const uint8_t* w_base[WI];
#pragma unroll
    for (int i = 0; i < WI; ++i) {
        const int at = (wave * WI + i) / 2, j = at % NB;
        int t = GATED ? n0 / 16 + at / NB * (NB / 2) + j % (NB / 2) : n0 / 16 + at;
        t = t < last_tile ? t : last_tile;
        w_base[i] = uniform_ptr(p.w[GATED ? j / (NB / 2) : 0] + (int64_t)t * p.blocks * 2048 + (wave * WI + i) % 2 * 1024);
    }
    const uint32_t w_off = lane * 16;
    uint32_t s_off;
    {
        const int r = wave * 64 + lane;
        s_off = (uint32_t)((m0 + r < p.M ? r : p.M - 1 - m0) * (int64_t)p.x_scales);
    }
    const uint8_t* s_base = p.xs + (int64_t)m0 * p.x_scales;

    auto fill = [&](int stage, int slot) __attribute__((always_inline)) {
        const uint8_t* xb = x_base + (int64_t)stage * 128;
#pragma unroll
        for (int i = 0; i < XI; ++i) copy16(lds0 + slot * XB + (wave * XI + i) * 1024, xb, x_off[i]);
#pragma unroll
        for (int i = 0; i < WI; ++i) copy16(ldsw + slot * WB + (wave * WI + i) * 1024, w_base[i] + (int64_t)stage * 2048, w_off);
    };
    auto fill_scales = [&](int four) __attribute__((always_inline)) {
        if (wave < SI) copy4(ldss + (four & 1) * BM * 4 + wave * 256, s_base + four * 4, s_off);
    };

    // Where this lane reads its operands of 16 rows or 16 weight rows.
    const int sw = c >> 1 & 7;
    const uint8_t* xr0 = lds + (wm * MB * 16 + c) * 128 + (g ^ sw) * 16;
    const uint8_t* xr1 = lds + (wm * MB * 16 + c) * 128 + ((g + 4) ^ sw) * 16;
    const uint8_t* wr = lds + 2 * XB + wn * NB * 2048 + lane * 16;
    const uint8_t* sr = lds + 2 * XB + 2 * WB + (wm * MB * 16 + c) * 4;
    typedef Block<EXACT, E8> B;

    f32x4 acc[NB][MB];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int m = 0; m < MB; ++m) acc[n][m] = f32x4{0, 0, 0, 0};
    B w[NB], x[2][2];
    uint32_t xs[2][2], ws[GATED ? 2 : 1];

    auto read_x = [&](int to, int slot, int m, int stage) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[to][i].load(xr0 + slot * XB + (m + i) * 2048, xr1 + slot * XB + (m + i) * 2048);
            xs[to][i] = *reinterpret_cast<const uint32_t*>(sr + (stage >> 2 & 1) * BM * 4 + (m + i) * 64);
        }
    };
    // The wavefront's weight rows lie in one block of 128.
    const int wt0 = GATED ? n0 / 16 + wn * (NB / 2) : n0 / 16 + wn * NB, wt = wt0 < last_tile ? wt0 : last_tile;
    const int nk = p.blocks;
    auto read_ws = [&](int stage) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < (GATED ? 2 : 1); ++i) ws[i] = weight_scale<E8>(p, i, wt, stage < nk ? stage : nk - 1);
    };
    auto products = [&](int from, int n, int m, int stage) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            mma_block(w[n], x[from][i], acc[n][m + i], ws[GATED ? n / (NB / 2) : 0], xs[from][i] >> (stage & 3) * 8 & 255);
    };
    auto step = [&](auto parity, int stage) __attribute__((always_inline)) {
        constexpr int S = decltype(parity)::value;
#pragma unroll
        for (int ph = 0; ph < PH - 1; ++ph) {
            read_x((ph & 1) ^ 1, S, 2 * ph + 2, stage);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < NB; ++n) products(ph & 1, n, 2 * ph, stage);
            __builtin_amdgcn_sched_barrier(0);
        }
        static_assert(PH % 2 == 0, "rows' blocks are read into either half in turn");
        __builtin_amdgcn_s_waitcnt(kWaitAll);
        asm volatile("s_barrier" ::: "memory");
        if (stage + 2 < nk) fill(stage + 2, S);
        if ((stage & 3) == 0 && stage + 4 < nk) fill_scales((stage >> 2) + 1);
        // Past the last stage this reads what the slot holds, for nothing.
        read_x(0, S ^ 1, 0, stage + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            products(1, n, MB - 2, stage);
            __builtin_amdgcn_sched_barrier(0);
            w[n].load(wr + (S ^ 1) * WB + n * 2048, wr + (S ^ 1) * WB + n * 2048 + 1024);
            __builtin_amdgcn_sched_barrier(0);
        }
        read_ws(stage + 1);
    };
    fill_scales(0);
    fill(0, 0);
    if (nk > 1) {
        fill(1, 1);
        __builtin_amdgcn_s_waitcnt(wait_vm(XI + WI));
    } else {
        __builtin_amdgcn_s_waitcnt(wait_vm(0));
    }
    asm volatile("s_barrier" ::: "memory");
#pragma unroll
    for (int n = 0; n < NB; ++n) w[n].load(wr + n * 2048, wr + n * 2048 + 1024);
    read_ws(0);
    read_x(0, 0, 0, 0);
    for (int stage = 0; stage < nk; stage += 2) {
        step(std::integral_constant<int, 0>(), stage);
        if (stage + 1 < nk) step(std::integral_constant<int, 1>(), stage + 1);
    }

    if constexpr (!CODES) {
        constexpr int N = GATED ? NB / 2 : NB;  // column blocks of the result a wavefront
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            const int row = m0 + (wm * MB + m) * 16 + c;
            if (row >= p.M) continue;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = GATED ? gate_value(acc[n][m][i], acc[n + NB - N][m][i], p.activation) : acc[n][m][i];
                store_row(static_cast<T*>(p.y) + (int64_t)row * p.N, n0 + (wn * N + n) * 16 + g * 4, p.N, v);
            }
        }
    } else {
        // Rows in 8 bits: the tile has all of a block's 128 columns.
        constexpr int N = NB / 2;
        static_assert(!CODES || (GATED && BN == 128), "a block of 128 a tile");
        float* top = reinterpret_cast<float*>(lds);                // [WN][BM]
        uint8_t* out = lds + WN * BM * 4;                          // [BM][144]
        __syncthreads();
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            float amax = 0.f;
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v = gate_value(acc[n][m][i], acc[n + N][m][i], p.activation);
                    if (n0 + (wn * N + n) * 16 + g * 4 + i >= p.N) v = 0.f;
                    acc[n][m][i] = v;
                    amax = fmaxf(amax, finite_magnitude(v));
                }
            amax = column_max(amax);
            if (g == 0) top[wn * BM + (wm * MB + m) * 16 + c] = amax;
        }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            const int r = (wm * MB + m) * 16 + c;
            float amax = top[r];
#pragma unroll
            for (int i = 1; i < WN; ++i) amax = fmaxf(amax, top[i * BM + r]);
            const uint32_t byte = fp8_scale_byte(amax);
            const float inv = fp8_scale_inverse(byte);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const f32x4 v = acc[n][m] * inv;
                *reinterpret_cast<uint32_t*>(out + r * 144 + (wn * N + n) * 16 + g * 4) = fp8_high(v[2], v[3], fp8_low(v[0], v[1]));
            }
            const int64_t blocks = fp8_blocks(p.N), per_row = fp8_scales(p.N);
            if (wn == 0 && m0 + r < p.M) {
                uint8_t* to = p.scales + (m0 + r) * per_row + n0 / 128;
                if (g == 0) to[0] = (uint8_t)byte;
                if (g > 0 && n0 + 128 >= p.N && n0 / 128 + g < per_row) to[g] = 0;  // past the blocks
            }
            if (m == MB - 1) {
                __syncthreads();
                for (int i = threadIdx.x; i < BM * 8; i += 64 * NW)
                    if (m0 + i / 8 < p.M)
                        *reinterpret_cast<u32x4*>(p.codes + ((m0 + i / 8) * blocks * 128 + n0 + i % 8 * 16)) =
                            *reinterpret_cast<const u32x4*>(out + i / 8 * 144 + i % 8 * 16);
            }
        }
    }
}

template <typename T, bool E8, bool GATED, int WM, int WN, int MB, int NB>
int tiles_run(const Fp8Params& p, hipStream_t st) {
    constexpr int BM = WM * MB * 16, BN = WN * NB * (GATED ? 8 : 16);
    const int64_t tm = (p.M + BM - 1) / BM, tn = (p.N + BN - 1) / BN;
    if (tm * tn > kMaxGrid / 2) return set_error(TT_UNSUPPORTED, "8-bit products: %lld tiles", (long long)(tm * tn));
    fp8_tiles_kernel<T, E8, GATED, WM, WN, MB, NB><<<(uint32_t)(tm * tn), 64 * WM * WN, 0, st>>>(p, (int)tm, (int)tn);
    return check_launch("8-bit products");
}

template <typename T, bool E8, bool GATED>
int tiles_shape(const Fp8Params& p, hipStream_t st) {
    if constexpr (std::is_same<T, float>::value)
        return tiles_run<T, E8, GATED, 2, 2, 4, 4>(p, st);
    else
        return tiles_run<T, E8, GATED, 2, 4, 8, 4>(p, st);
}

template <bool E8, bool GATED>
int tiles_typed(int64_t dtype, const Fp8Params& p, hipStream_t st) {
    if constexpr (GATED)
        if (p.codes) return tiles_shape<Codes, E8, GATED>(p, st);
    if (dtype == TT_F32) return tiles_shape<float, E8, GATED>(p, st);
    return dtype == TT_BF16 ? tiles_shape<__bf16, E8, GATED>(p, st) : tiles_shape<_Float16, E8, GATED>(p, st);
}

}  // namespace

int fp8_tiles(int64_t dtype, bool e8, bool gated, const Fp8Params& p, hipStream_t st) {
    if (gated) return e8 ? tiles_typed<true, true>(dtype, p, st) : tiles_typed<false, true>(dtype, p, st);
    return e8 ? tiles_typed<true, false>(dtype, p, st) : tiles_typed<false, false>(dtype, p, st);
}

}  // namespace tt
