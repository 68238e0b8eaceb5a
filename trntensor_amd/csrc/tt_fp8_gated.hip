// The gated half of a feed-forward block in 8 bits on workgroup tiles.
#include "tt_fp8_tiles.hpp"

namespace tt {

namespace {

template <typename T, bool E8>
int tiles_of(int which, const Fp8Params& p, hipStream_t st) {
    // Raw results of these two would have a block's 128 columns: written as codes at once.
    if constexpr (!std::is_same<T, Raw>::value) {
        if (which == 0) return tiles_run<T, E8, true, 2, 4, 8, 4, 2>(p, st);
        if (which == 1) return tiles_run<T, E8, true, 2, 4, 4, 4, 3>(p, st);
    }
    switch (which) {
        case 2:
            return tiles_run<T, E8, true, 2, 2, 4, 4, 4>(p, st);
        case 3:
            return tiles_run<T, E8, true, 2, 2, 2, 4, 4>(p, st);
        default:
            return tiles_run<T, E8, true, 2, 2, 2, 2, 5>(p, st);
    }
}

template <bool E8>
int exact_of(int which, const Fp8Params& p, hipStream_t st) {
    if (which == 0) return tiles_run<Single, E8, true, 2, 2, 4, 4, 2>(p, st);
    return tiles_run<Single, E8, true, 2, 2, 2, 2, 4>(p, st);
}

// 32-bit products of the 8-bit matrix instructions into rows of 8 bits: one workgroup
// 2048 elements of a row, blocks whose scale they do not decide computed again.
template <bool E8>
__global__ __launch_bounds__(256) void gated_round_kernel(Fp8Params p, int pieces) {
    const int row = blockIdx.x / pieces, lane = threadIdx.x & 63;
    const int col = (int)(blockIdx.x % pieces) * 2048 + (int)threadIdx.x * 8;
    const int blocks = (p.N + 127) / 128;
    const float* from = static_cast<const float*>(p.y) + (int64_t)row * p.N;
    Eight<float> x;
    x.load(from, col, p.N);
    float v[8], amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = x.get(i);
        amax = fmaxf(amax, finite_magnitude(v[i]));
    }
    amax = max_of_16(amax);
    if (__any(near_border(amax))) {
        float again = 0.f;
        // At most 16 values of a wavefront's four blocks.
        int left = 16;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint64_t which = __ballot(near_border(amax) && finite_magnitude(v[i]) >= amax * kCandidate);
            for (; which != 0 && left > 0; which &= which - 1, --left) {
                const int l = __builtin_ctzll(which);
                float sum[2];
                exact_parts<E8, 8>(p, row, __builtin_amdgcn_readlane(col, l) + i, lane, 64, sum);
                const float h = exact_gated(sum, p.activation);
                if (lane / 16 == l / 16) again = fmaxf(again, h);
            }
        }
        if (near_border(amax) && left > 0 && again > 0.f) amax = decided(amax, again);
    }
    fp8_store8(v, amax, col, blocks, p.codes + (int64_t)row * blocks * 128, p.scales + (int64_t)row * ((blocks + 3) / 4 * 4));
}

// Tiles that have all of a block's 128 columns.
template <bool E8>
int codes_of(int which, const Fp8Params& p, hipStream_t st) {
    switch (which) {
        case 0:
            return tiles_run<Codes, E8, true, 2, 4, 8, 4, 2>(p, st);
        case 1:
            return tiles_run<Codes, E8, true, 2, 4, 4, 4, 3>(p, st);
        case 2:
            return tiles_run<Codes, E8, true, 1, 4, 4, 4, 3>(p, st);
        default:
            return tiles_run<Codes, E8, true, 1, 4, 2, 4, 4>(p, st);
    }
}

}  // namespace

// us a step of 256 workgroups, as in fp8_tiles_cost (a gated tile of N columns reads
// and multiplies what one of 2 N does). Tiles that write codes have 128 columns,
// and take longer a step from 64 rows down: 64 x 128 0.7, 32 x 128 0.6.
double fp8_gated_tiles_cost(const Fp8Params& p, int kind, int* which) {
    const int shapes[5][2] = {{256, 128}, {128, 128}, {128, 64}, {64, 64}, {64, 32}};
    const double steps[5] = {1.38, 0.95, 0.52, 0.345, 0.225};
    const int code_shapes[4] = {256, 128, 64, 32};
    const double code_steps[4] = {1.38, 0.95, 0.7, 0.6};
    double best = 0;
    if (kind == kExact) {
        const double big = tiles_cost(p, 128, 64, 1.0), small = tiles_cost(p, 64, 32, 0.4);
        *which = big < small ? 0 : 1;
        best = big < small ? big : small;
    } else if (kind == kCodes) {
        for (int i = 0; i < 4; ++i) {
            const double cost = tiles_cost(p, code_shapes[i], 128, code_steps[i]);
            if (i == 0 || cost < best) best = cost, *which = i;
        }
    } else {
        const int first = kind == kRaw ? 2 : 0;
        for (int i = first; i < 5; ++i) {
            const double cost = tiles_cost(p, shapes[i][0], shapes[i][1], steps[i]);
            if (i == first || cost < best) best = cost, *which = i;
        }
    }
    return best * p.blocks;
}

int fp8_gated_tiles(int kind, bool e8, int which, const Fp8Params& p, hipStream_t st) {
    if (kind == kExact) return e8 ? exact_of<true>(which, p, st) : exact_of<false>(which, p, st);
    if (kind == kCodes) return e8 ? codes_of<true>(which, p, st) : codes_of<false>(which, p, st);
    if (kind == kRaw) return e8 ? tiles_of<Raw, true>(which, p, st) : tiles_of<Raw, false>(which, p, st);
    return e8 ? tiles_of<Half, true>(which, p, st) : tiles_of<Half, false>(which, p, st);
}

int fp8_gated_round(bool e8, const Fp8Params& p, hipStream_t st) {
    const int pieces = (p.N + 2047) / 2048;
    if (e8)
        gated_round_kernel<true><<<(uint32_t)p.M * pieces, 256, 0, st>>>(p, pieces);
    else
        gated_round_kernel<false><<<(uint32_t)p.M * pieces, 256, 0, st>>>(p, pieces);
    return check_launch("tt_fp8_gated_matmul");
}

}  // namespace tt
