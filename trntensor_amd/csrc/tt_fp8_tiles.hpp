// Products of many rows in 8 bits with 8-bit weights, and the gated block on
// two of them (tt_fp8_tiles.hip, tt_fp8_gated.hip): workgroup tiles whose operands
// are copied global -> LDS by direct loads.
//
// A workgroup has WM x WN wavefronts of MB x NB blocks of 16 x 16. A stage is one
// block of 128 columns: rows of x as eight 16-byte pieces, piece p of row r at
// position p ^ (r / 2 % 8) so that 16 lanes' reads cover 256 bytes, and weight
// tiles as they are packed. NS stages are held; a step multiplies one of them:
//   the rows' blocks one at a time, the next one being read from LDS meanwhile;
//   before the last one, all reads of the stage are done and the next stage has
//   arrived: one barrier, behind which this stage's slot is filled again (NS
//   steps ahead) and the next stage's weights and first rows are read while the
//   last block is multiplied.
// The rows' scales come along with each stage, those of the four blocks that its
// own belongs to, 4 bytes a row. No branch stands among the products: it would let
// the compiler gather them behind it, and all operands in registers before it. What
// bounds large calls is the matrix units' time (75% of it busy at 4096 x 8192 x 8192,
// 2.7 PFLOP/s) and what a wavefront issues between two products.
#pragma once

#include <type_traits>

#include "tt_fp8_block.hpp"

namespace tt {

namespace {

__device__ __forceinline__ unsigned lds_address(const void* p) {
    return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// Values that all lanes share, for scalar registers, with the five wait states from a
// vector instruction that writes one to a load that reads it: the compiler does not
// keep them to loads in assembly.
__device__ __forceinline__ unsigned uniform(unsigned x) {
    unsigned r = (unsigned)__builtin_amdgcn_readfirstlane((int)x);
    asm volatile("s_nop 4" : "+s"(r));
    return r;
}
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
    const uint64_t v = (uint64_t)(uintptr_t)p;
    return (const uint8_t*)(uintptr_t)((uint64_t)uniform((unsigned)v) | (uint64_t)uniform((unsigned)(v >> 32)) << 32);
}

// Direct loads, 16 and 4 bytes a lane, to LDS address `to` + 16 or 4 * lane, from base
// + offset; `to` and base are scalars. They are assembly so that the compiler does not
// take them for writes that every LDS read has to wait for; the kernel's own waits
// and barriers order them. Nothing else here uses M0, and all lanes are on. The
// no-operation is the wait state from a write of M0 to its use.
__device__ __forceinline__ void copy16(unsigned to, const uint8_t* base, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(to), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void copy4(unsigned to, const uint8_t* base, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" : : "s"(to), "v"(offset), "s"(base) : "memory", "m0");
}

// s_waitcnt immediates: vmcnt in bits 3:0 and 15:14, expcnt 6:4 (7: no wait), lgkmcnt 11:8.
constexpr int wait_vm(int n) { return (n & 15) | (n >> 4) << 14 | 0xf70; }
constexpr int kWaitLds = ~0xf00;  // and lgkmcnt(0)

// What the result is written as.
struct Half {};    // bfloat16 or float16, as the call says
struct Single {};  // float32, of exact sums
struct Raw {};     // float32, of the 8-bit matrix instructions' sums
struct Codes {};   // rows in 8 bits

template <typename T, bool E8, bool GATED, int WM, int WN, int MB, int NB, int NS>
__global__ __launch_bounds__(64 * WM * WN, 2) void fp8_tiles_kernel(Fp8Params p, int tiles_m, int tiles_n) {
    constexpr bool CODES = std::is_same<T, Codes>::value, EXACT = std::is_same<T, Single>::value;
    constexpr int NW = WM * WN, BM = WM * MB * 16;
    constexpr int NT = WN * NB;                          // weight tiles of 16 rows a stage
    constexpr int BN = GATED ? NT * 8 : NT * 16;         // columns of the result
    constexpr int XB = BM * 128, WB = NT * 2048, STAGE = XB + WB;  // bytes
    constexpr int XI = XB / 1024 / NW, WI = WB / 1024 / NW;  // direct loads a wavefront a stage
    constexpr int SI = (BM + 63) / 64;                   // wavefronts that load the rows' scales
    constexpr int SB = SI * 256;                         // bytes of a four of them
    constexpr int FOURS = 4;                             // of them held
    constexpr int GM = GATED ? 2 : 1;                    // weight matrices
    constexpr int WS = E8 ? FOURS : 16;                  // scales held of each: fours of bytes, or floats, of 64 tiles
    constexpr int PER = XI + WI + 1;                     // direct loads a wavefront a stage
    constexpr bool TWICE = NS >= 4;                      // registers hold the operands of two stages
    constexpr bool FLOATS = !E8 && !EXACT;
    constexpr int AHEAD = NS == 2 && !FLOATS ? 1 : 0;    // stages that lines are asked of L2 before their direct loads
    static_assert(XI * 1024 * NW == XB && WI * 1024 * NW == WB && NW >= SI + GM && MB % 2 == 0 && NB % 2 == 0, "tile");
    // The stages held belong to at most FOURS fours.
    static_assert(NS >= 2 && NS <= 9 && (NS - 1) * PER < 64, "stages");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[NS * STAGE + FOURS * SB + GM * WS * 256 + (AHEAD ? NW * 256 : 0)];
    const unsigned lds0 = uniform(lds_address(lds)), ldss = lds0 + NS * STAGE, ldsw = ldss + FOURS * SB;

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
    const uint8_t* x_base = uniform(p.x + m0 * pitch);
    uint32_t x_off[XI];
#pragma unroll
    for (int i = 0; i < XI; ++i) {
        const int r = (wave * XI + i) * 8 + (lane >> 3);
        const int row = m0 + r < p.M ? r : p.M - 1 - m0;
        x_off[i] = (uint32_t)(row * pitch) + (((lane & 7) ^ (r >> 1 & 7)) * 16);
    }
    const int last_tile = (p.N + 15) / 16 - 1;
    // A wavefront's weight tiles are of one matrix, or half of them of either.
    constexpr int WT = WI / 2, MATS = GATED && WT > NB / 2 ? 2 : 1, WE = WT / MATS;  // tiles, matrices, tiles of each
    static_assert(WI % 2 == 0 && (!GATED || (MATS == 1 ? NB / 2 % WT == 0 : WT == NB)), "tiles of one matrix");
    auto weight_tile = [&](int at) __attribute__((always_inline)) {
        const int t = GATED ? n0 / 16 + at / NB * (NB / 2) + at % NB % (NB / 2) : n0 / 16 + at;
        return t < last_tile ? t : last_tile;
    };
    const uint8_t* w_base[MATS];
    uint32_t w_off[WT];  // at most 15 tiles on
#pragma unroll
    for (int i = 0; i < MATS; ++i) {
        const int at = wave * WT + i * WE, t0 = weight_tile(at);
        w_base[i] = uniform(p.w[GATED ? at % NB / (NB / 2) : 0] + (int64_t)t0 * p.blocks * 2048);
#pragma unroll
        for (int e = 0; e < WE; ++e) w_off[i * WE + e] = (uint32_t)(weight_tile(at + e) - t0) * (uint32_t)p.blocks * 2048 + lane * 16;
    }
    // The first wavefronts load the rows' scales, a row a lane; the others those
    // of the weights, a tile a lane (as often as there are more lanes).
    const bool of_rows = wave < SI;
    const int matrix = (wave - SI) & (GM - 1);
    uint32_t s_off;
    const uint8_t* s_base;
    if (of_rows) {
        const int r = wave * 64 + lane;
        s_base = p.xs + (int64_t)m0 * p.x_scales;
        s_off = (uint32_t)((m0 + r < p.M ? r : p.M - 1 - m0) * (int64_t)p.x_scales);
    } else {
        const int pitch_ws = E8 ? p.x_scales : p.blocks * 4, t0 = n0 / 16, t = t0 + lane % (NT / GM);
        s_base = p.ws[matrix] + (int64_t)(t0 / 8) * pitch_ws;
        s_off = (uint32_t)(((t < last_tile ? t : last_tile) / 8 - t0 / 8) * pitch_ws);
    }
    s_base = uniform(s_base);
    // Fours of bytes lie at the multiples of four, floats at four times their stage.
    const bool fours = of_rows || E8;
    const uint32_t s_held = fours ? 4 * FOURS - 4 : WS - 1, s_shift = of_rows ? 6 + (SI > 1) + (SI > 2) : fours ? 6 : 8;
    static_assert(SI == 1 || SI == 2 || SI == 4, "bytes of a four: 256 SI");
    const unsigned s_to = of_rows ? ldss + wave * 256 : ldsw + matrix * WS * 256;

    // Direct loads [from, to) of a stage, whose place in LDS is `slot`. Past the last
    // stage they are of that once more, for nothing: what stands between two products
    // counts, and a mask is four scalar instructions a load. With it, a base for each
    // load and signed and 64-bit arithmetic, 4096 x 8192 x 8192 took 217 us (now 210), with
    // float scales 231 (224), 1024 x 4096 x 4096 with them 24.7 (22.0), 2048 x 16384 x 4096
    // gated 222 (215).
    const unsigned x_to = lds0 + wave * XI * 1024, w_to = lds0 + XB + wave * WI * 1024;
    auto fill = [&](int stage, int slot, int from, int to) __attribute__((always_inline)) {
        const uint32_t at = stage < p.blocks ? stage : p.blocks - 1;
        const uint8_t* x = x_base + at * 128;
#pragma unroll
        for (int i = from; i < to; ++i) {
            if (i < XI)
                copy16(x_to + slot + i * 1024, x, x_off[i]);
            else if (i < XI + WI)
                copy16(w_to + slot + (i - XI) * 1024, w_base[(i - XI) / 2 / WE] + (at * 2048 + (i - XI) % 2 * 1024), w_off[(i - XI) / 2]);
            else
                copy4(s_to + ((at & s_held) << s_shift), s_base + (fours ? at & ~3u : at * 4), s_off);
        }
    };

    // Two stages in LDS leave a direct load one step to arrive in, which is less
    // than a line takes that is not in L2: each line is asked for a step earlier
    // by one of the workgroups that share it (four of the same weights, eight or
    // more of the same rows, on one XCD), as one word of it to a place nobody reads.
    // A wavefront whose turn it is not asks for one line that it has. 4096 x 8192 x 8192
    // takes 204 us with it, 217 without; with float scales, whose steps are longer, it
    // costs what it saves (242 / 239).
    const uint8_t* line = x_base;
    uint32_t line_off = 0;
    int line_step = 0;
    if constexpr (AHEAD > 0) {
        constexpr int XL = BM / 64, WL = NT / 4;  // wavefronts that have all lines
        static_assert(XL + WL <= NW && (!GATED || NB == 4), "a line a lane, of one matrix a wavefront");
        if (wave < XL) {
            const int r = wave * 64 + lane;
            if (rest / high % XL == wave) {
                line_off = (uint32_t)((m0 + r < p.M ? r : p.M - 1 - m0) * pitch);
                line_step = 128;
            }
        } else if (wave < XL + WL && rest % high % WL == wave - XL) {
            // Four neighbouring tiles, gated ones of the one matrix or of the other.
            const int q = wave - XL, t0 = n0 / 16 + (GATED ? q / 2 : q) * 4, t = t0 + lane / 16;
            const int least = t0 < last_tile ? t0 : last_tile;
            line = uniform(p.w[GATED ? q & 1 : 0] + (int64_t)least * p.blocks * 2048);
            line_off = (uint32_t)((t < last_tile ? t : last_tile) - least) * (uint32_t)p.blocks * 2048 + lane % 16 * 128;
            line_step = 2048;
        }
    }
    auto ask = [&](int stage) __attribute__((always_inline)) {
        const int s = stage < p.blocks ? stage : p.blocks - 1;
        copy4(ldsw + GM * WS * 256 + wave * 256, line + (uint32_t)s * (uint32_t)line_step, line_off);
    };

    // Where this lane reads its operands of 16 rows or 16 weight rows.
    const int sw = c >> 1 & 7;
    const uint8_t* xr0 = lds + (wm * MB * 16 + c) * 128 + (g ^ sw) * 16;
    const uint8_t* xr1 = lds + (wm * MB * 16 + c) * 128 + ((g + 4) ^ sw) * 16;
    const uint8_t* wr = lds + XB + wn * NB * 2048 + lane * 16;
    const uint8_t* sr = lds + NS * STAGE + (wm * MB * 16 + c) * 4;
    const uint8_t* wsr = lds + NS * STAGE + FOURS * SB + wn * (NB / GM) * 4;  // the wavefront's weights lie in one block of 128

    f32x4 acc[NB][MB];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int m = 0; m < MB; ++m) acc[n][m] = f32x4{0, 0, 0, 0};
    const int nk = p.blocks;
    // With float scales a block's sum is multiplied when DEPTH products after it are on
    // their way: two 26.0 us for 1024 x 4096 x 4096, one 27.6, three 26.3; 249 / 256 /
    // 247 for 2048 x 16384 x 4096 gated, with one sum less to hold than three.
    constexpr int DEPTH = 2;
    typedef Block<EXACT, E8> B;
    f32x4 sum[DEPTH];
    auto scaled = [&](int at, const uint32_t (&ws)[GM]) __attribute__((always_inline)) {
        acc[at % NB][at / NB] += __uint_as_float(ws[GATED ? at % NB / (NB / 2) : 0]) * sum[at % DEPTH];
    };
    auto last_scaled = [&](const uint32_t (&ws)[GM]) __attribute__((always_inline)) {
        if constexpr (FLOATS)
#pragma unroll
            for (int i = DEPTH; i > 0; --i) scaled(MB * NB - i, ws);
    };
    auto product = [&](int n, int m, const B& w, const B& x, const uint32_t (&ws)[GM], uint32_t sb) __attribute__((always_inline)) {
        if constexpr (FLOATS) {
            const int at = m * NB + n;
            const f32x4 next = block_sum(w, x, sb);
            __builtin_amdgcn_sched_barrier(0);
            if (at >= DEPTH) scaled(at - DEPTH, ws);
            __builtin_amdgcn_sched_barrier(0);
            sum[at % DEPTH] = next;
        } else {
            mma_block(w, x, acc[n][m], ws[GATED ? n / (NB / 2) : 0], sb);
        }
    };
    auto read_x = [&](B& x, uint32_t& xs, int slot, int m, int stage) __attribute__((always_inline)) {
        x.load(xr0 + slot + m * 2048, xr1 + slot + m * 2048);
        xs = *reinterpret_cast<const uint32_t*>(sr + ((stage >> 2) & (FOURS - 1)) * SB + m * 64);
    };
    auto read_w = [&](B& w, int slot, int n) __attribute__((always_inline)) {
        w.load(wr + slot + n * 2048, wr + slot + n * 2048 + 1024);
    };
    auto read_ws = [&](uint32_t (&ws)[GM], int stage) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < GM; ++i) ws[i] = *reinterpret_cast<const uint32_t*>(wsr + (i * WS + ((E8 ? stage >> 2 : stage) & (WS - 1))) * 256);
    };
    auto take_ws = [&](uint32_t (&ws)[GM], int stage) __attribute__((always_inline)) {
        if constexpr (E8)
#pragma unroll
            for (int i = 0; i < GM; ++i) ws[i] = ws[i] >> (stage & 3) * 8 & 255;
    };
    int slot = 0, last = (NS - 1) * STAGE;
    if constexpr (!TWICE) {
        constexpr int XR = MB % 4 == 0 ? 4 : 2, LEAD = XR / 2;  // blocks of rows in registers, and read ahead
        // Products that a stage's direct loads are spread over, some of them behind
        // the barrier and the rest in the next step: half of them 204 us for 4096 x 8192 x
        // 8192, 7 of 16 210, 9 207, 5 217; with float scales 228, 225, 229 and 225.
        constexpr int SPREAD = MB * NB * (FLOATS ? 7 : 8) / 16, LATE = PER * (LEAD * NB < SPREAD ? LEAD * NB : SPREAD) / SPREAD;
        B w[NB], x[XR];
        uint32_t xs[XR], ws[GM], next_ws[GM];
        auto step = [&](int stage) __attribute__((always_inline)) {
            const int next = slot == (NS - 1) * STAGE ? 0 : slot + STAGE;
#pragma unroll
            for (int m = 0; m < MB; ++m) {
                if (m == MB - LEAD) {
                    // The next stage was filled before NS - 2 others.
                    __builtin_amdgcn_s_waitcnt(wait_vm((NS - 2) * PER + (AHEAD > 0)) & kWaitLds);
                    asm volatile("s_barrier" ::: "memory");
                }
                const uint32_t sb = xs[m % XR] >> (stage & 3) * 8 & 255;
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    product(n, m, w[n], x[m % XR], ws, sb);
                    __builtin_amdgcn_sched_barrier(0);
                    // Past the last stage these read what the slot holds, for nothing.
                    if (n == 0) {
                        if (m < MB - LEAD)
                            read_x(x[(m + LEAD) % XR], xs[(m + LEAD) % XR], slot, m + LEAD, stage);
                        else
                            read_x(x[(m + LEAD) % XR], xs[(m + LEAD) % XR], next, m + LEAD - MB, stage + 1);
                    }
                    if (m == MB - 1) read_w(w[n], next, n);
                    if (m == MB - 1 && n == 0) read_ws(next_ws, stage + 1);
                    const int at = ((m - (MB - LEAD) + MB) % MB) * NB + n;  // products since the barrier
                    const bool before = m < MB - LEAD;
                    if (at < SPREAD) fill(stage + NS - before, before ? last : slot, PER * at / SPREAD, PER * (at + 1) / SPREAD);
                    if constexpr (AHEAD > 0)
                        if (at == SPREAD) ask(stage + NS - before + AHEAD);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            last_scaled(ws);
#pragma unroll
            for (int i = 0; i < GM; ++i) ws[i] = next_ws[i];
            take_ws(ws, stage + 1);
            last = slot;
            slot = next;
        };
#pragma unroll
        for (int s = 0; s < NS; ++s) fill(s, s * STAGE, 0, s < NS - 1 ? PER : LATE);
        __builtin_amdgcn_s_waitcnt(wait_vm((NS - 2) * PER + LATE));
        asm volatile("s_barrier" ::: "memory");
#pragma unroll
        for (int n = 0; n < NB; ++n) read_w(w[n], 0, n);
        read_ws(ws, 0);
        take_ws(ws, 0);
#pragma unroll
        for (int m = 0; m < LEAD; ++m) read_x(x[m], xs[m], 0, m, 0);
        for (int stage = 0; stage < nk; ++stage) step(stage);
    } else {
        B w[2][NB], x[2][MB];
        uint32_t xs[2][MB], ws[2][GM];
        auto step = [&](auto parity, int stage) __attribute__((always_inline)) {
            constexpr int P = decltype(parity)::value;
            const int next = slot == (NS - 1) * STAGE ? 0 : slot + STAGE;
            take_ws(ws[P], stage);
#pragma unroll
            for (int m = 0; m < MB; ++m) {
                const uint32_t sb = xs[P][m] >> (stage & 3) * 8 & 255;
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    product(n, m, w[P][n], x[P][m], ws[P], sb);
                    __builtin_amdgcn_sched_barrier(0);
                    // The next stage's operands (past the last stage, what the slot holds).
                    const int at = m * NB + n;
                    if (at == 0) read_ws(ws[P ^ 1], stage + 1);
                    if (at < NB) read_w(w[P ^ 1][at], next, at);
                    if (at >= MB * NB - MB) read_x(x[P ^ 1][at - (MB * NB - MB)], xs[P ^ 1][at - (MB * NB - MB)], next, at - (MB * NB - MB), stage + 1);
                    fill(stage + NS - 1, last, PER * at / (MB * NB), PER * (at + 1) / (MB * NB));
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            last_scaled(ws[P]);
            // The stage after the next was filled before NS - 3 others.
            __builtin_amdgcn_s_waitcnt(wait_vm((NS - 3) * PER));
            asm volatile("s_barrier" ::: "memory");
            last = slot;
            slot = next;
        };
#pragma unroll
        for (int s = 0; s < NS - 1; ++s) fill(s, s * STAGE, 0, PER);
        __builtin_amdgcn_s_waitcnt(wait_vm((NS - 3) * PER));
        asm volatile("s_barrier" ::: "memory");
#pragma unroll
        for (int n = 0; n < NB; ++n) read_w(w[0][n], 0, n);
        read_ws(ws[0], 0);
#pragma unroll
        for (int m = 0; m < MB; ++m) read_x(x[0][m], xs[0][m], 0, m, 0);
        int stage = 0;
        for (; stage + 1 < nk; stage += 2) {
            step(std::integral_constant<int, 0>(), stage);
            step(std::integral_constant<int, 1>(), stage + 1);
        }
        if (stage < nk) step(std::integral_constant<int, 0>(), stage);
    }
    __builtin_amdgcn_s_waitcnt(wait_vm(0));

    if constexpr (!CODES) {
        // Through LDS, so that what is stored together is rows' whole lines: stored from
        // the accumulators, 32 bytes of a row each, a call of one tile of 256 x 256 and
        // one block of columns took 11.3 us, so 4.9.
        constexpr int N = GATED ? NB / 2 : NB;  // column blocks of the result a wavefront
        typedef typename std::conditional<std::is_same<T, Half>::value, uint16_t, uint32_t>::type E;
        constexpr int PITCH = BN * sizeof(E) + 16, PIECES = BN * sizeof(E) / 16, EACH = 16 / sizeof(E);
        static_assert(BM * PITCH <= (int)sizeof lds, "the result fits in LDS");
        __syncthreads();
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
            for (int n = 0; n < N; ++n) {
                E e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float v = GATED ? gate_value(acc[n][m][i], acc[n + NB - N][m][i], p.activation) : acc[n][m][i];
                    if constexpr (sizeof(E) == 4)
                        e[i] = __float_as_uint(v);
                    else
                        e[i] = p.bf16 ? __builtin_bit_cast(uint16_t, (__bf16)v) : __builtin_bit_cast(uint16_t, (_Float16)v);
                }
                __builtin_memcpy(__builtin_assume_aligned(lds + ((wm * MB + m) * 16 + c) * PITCH + ((wn * N + n) * 16 + g * 4) * sizeof(E), 8), e, sizeof e);
            }
        __syncthreads();
        for (int i = threadIdx.x; i < BM * PIECES; i += 64 * NW) {
            const int row = m0 + i / PIECES, col = n0 + i % PIECES * EACH;
            if (row >= p.M || col >= p.N) continue;
            const E* from = reinterpret_cast<const E*>(lds + i / PIECES * PITCH) + i % PIECES * EACH;
            E* to = static_cast<E*>(p.y) + (int64_t)row * p.N + col;
            if (col + EACH <= p.N) {
                E e[EACH];
                __builtin_memcpy(e, __builtin_assume_aligned(from, 16), sizeof e);
                __builtin_memcpy(to, e, sizeof e);
            } else {
                for (int j = 0; j < p.N - col; ++j) to[j] = from[j];
            }
        }
    } else {
        // Rows in 8 bits: the tile has all of a block's 128 columns.
        constexpr int N = NB / 2;
        static_assert(!CODES || (GATED && BN == 128), "a block of 128 a tile");
        constexpr int LIST = 64;
        float* top = reinterpret_cast<float*>(lds);                // [WN][BM]
        float* again = top + WN * BM;                              // [BM], largest values computed again
        float* parts = again + BM;                                 // [NW][2]
        int* list = reinterpret_cast<int*>(parts + 2 * NW);        // their places, and how many
        uint8_t* out = reinterpret_cast<uint8_t*>(list + LIST + 4);  // [BM][144]
        static_assert(!CODES || (WN + 1) * BM * 4 + (2 * NW + LIST + 4) * 4 + BM * 144 <= (int)sizeof lds, "LDS");
        __syncthreads();
        for (int i = threadIdx.x; i < BM; i += 64 * NW) again[i] = 0.f;
        if (threadIdx.x == 0) list[LIST] = 0;
        auto values = [&](auto activation) __attribute__((always_inline)) {
#pragma unroll
            for (int m = 0; m < MB; ++m)
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        acc[n][m][i] = gate_value<decltype(activation)::value>(acc[n][m][i], acc[n + N][m][i]);
        };
        if (p.activation == 0)
            values(std::integral_constant<int, 0>());
        else
            values(std::integral_constant<int, 1>());
        if (n0 + 128 > p.N) {
#pragma unroll
            for (int m = 0; m < MB; ++m)
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (n0 + (wn * N + n) * 16 + g * 4 + i >= p.N) acc[n][m][i] = 0.f;
        }
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            float amax = 0.f;  // NaN has no part in it
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(acc[n][m][i]));
            if (__any(amax == INFINITY)) {  // infinities become NaN
                amax = 0.f;
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (fabsf(acc[n][m][i]) == INFINITY) acc[n][m][i] = NAN;
                        amax = fmaxf(amax, fabsf(acc[n][m][i]));
                    }
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
            if (near_border(amax) && m0 + r < p.M) {
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (fabsf(acc[n][m][i]) >= amax * kCandidate) {
                            const int at = atomicAdd(&list[LIST], 1);
                            if (at < LIST) list[at] = r * 128 + (wn * N + n) * 16 + g * 4 + i;
                        }
            }
        }
        __syncthreads();
        // More than the list holds (inputs that are all alike) stay as they are.
        const int count = __builtin_amdgcn_readfirstlane(list[LIST]);
        // (Mostly there are none or one: the whole workgroup takes each.)
        if (count <= LIST)
            for (int e = 0; e < count; ++e) {
                const int at = __builtin_amdgcn_readfirstlane(list[e]);
                float sum[2];
                exact_parts<E8, 1>(p, m0 + at / 128, n0 + at % 128, threadIdx.x, 64 * NW, sum);
                if (lane == 0) parts[2 * wave] = sum[0], parts[2 * wave + 1] = sum[1];
                __syncthreads();
                if (threadIdx.x == 0) {
#pragma unroll
                    for (int i = 1; i < NW; ++i) sum[0] += parts[2 * i], sum[1] += parts[2 * i + 1];
                    again[at / 128] = fmaxf(again[at / 128], exact_gated(sum, p.activation));
                }
                __syncthreads();
            }
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            const int r = (wm * MB + m) * 16 + c;
            float amax = top[r];
#pragma unroll
            for (int i = 1; i < WN; ++i) amax = fmaxf(amax, top[i * BM + r]);
            if (near_border(amax) && count <= LIST && again[r] > 0.f) amax = decided(amax, again[r]);
            const uint32_t byte = fp8_scale_byte(amax);
            const float inv = fp8_scale_inverse(byte);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const f32x4 v = acc[n][m] * inv;  // 448 at most, and 2^-11 of it where computed again
                const uint32_t low = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
                *reinterpret_cast<uint32_t*>(out + r * 144 + (wn * N + n) * 16 + g * 4) =
                    (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], (int)low, true);
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

template <typename T, bool E8, bool GATED, int WM, int WN, int MB, int NB, int NS>
int tiles_run(const Fp8Params& p, hipStream_t st) {
    constexpr int BM = WM * MB * 16, BN = WN * NB * (GATED ? 8 : 16);
    const int64_t tm = (p.M + BM - 1) / BM, tn = (p.N + BN - 1) / BN;
    if (tm * tn > kMaxGrid / 2) return set_error(TT_UNSUPPORTED, "8-bit products: %lld tiles", (long long)(tm * tn));
    fp8_tiles_kernel<T, E8, GATED, WM, WN, MB, NB, NS><<<(uint32_t)(tm * tn), 64 * WM * WN, 0, st>>>(p, (int)tm, (int)tn);
    return check_launch("8-bit products");
}

// Steps of 256 workgroups that tiles of bm x bn take, times what a step takes.
inline double tiles_cost(const Fp8Params& p, int bm, int bn, double step) {
    const int64_t tiles = (int64_t)((p.M + bm - 1) / bm) * ((p.N + bn - 1) / bn);
    return (double)((tiles + 255) / 256) * step;
}

}  // namespace
}  // namespace tt
