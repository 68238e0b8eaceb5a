// Products of rows in 8 bits with 8-bit weights on workgroup tiles.
#include "tt_fp8_tiles.hpp"

namespace tt {

namespace {

template <typename T, bool E8>
int tiles_of(int which, const Fp8Params& p, hipStream_t st) {
    switch (which) {
        case 0:
            return tiles_run<T, E8, false, 2, 4, 8, 4, 2>(p, st);
        case 1:
            return tiles_run<T, E8, false, 2, 4, 4, 4, 3>(p, st);
        case 2:
            return tiles_run<T, E8, false, 2, 2, 4, 4, 4>(p, st);
        case 3:
            return tiles_run<T, E8, false, 2, 2, 2, 4, 4>(p, st);
        default:
            return tiles_run<T, E8, false, 2, 2, 2, 2, 5>(p, st);
    }
}

template <bool E8>
int exact_of(int which, const Fp8Params& p, hipStream_t st) {
    if (which == 0) return tiles_run<Single, E8, false, 2, 2, 4, 4, 2>(p, st);
    return tiles_run<Single, E8, false, 2, 2, 2, 2, 4>(p, st);
}

}  // namespace

// us a step of 256 workgroups (K = 4096, 16-bit results): 256 x 256 1.38, 128 x 256
// 0.95, 128 x 128 0.52, 64 x 128 0.345, 64 x 64 0.225; a tile that needs fewer
// rounds of workgroups wins although it takes longer a step: 4096 x 8192 x 8192
// 209 / 247 / 327 / 395 / 535, 2048 x 4096 x 4096 47 / 35 / 37 / 51 / 71, 1024 rows
// 46 / 29 / 21 / 27 / 40, 512 rows 46 / 28 / 19 / 15 / 22, 256 rows 45 / 28 / 18 / 14 / 12.
double fp8_tiles_cost(const Fp8Params& p, bool exact, int* which) {
    const int shapes[5][2] = {{256, 256}, {128, 256}, {128, 128}, {64, 128}, {64, 64}};
    const double steps[5] = {1.38, 0.95, 0.52, 0.345, 0.225};
    double best = 0;
    if (exact) {
        const double big = tiles_cost(p, 128, 128, 1.0), small = tiles_cost(p, 64, 64, 0.4);
        *which = big < small ? 0 : 1;
        best = big < small ? big : small;
    } else {
        for (int i = 0; i < 5; ++i) {
            const double cost = tiles_cost(p, shapes[i][0], shapes[i][1], steps[i]);
            if (i == 0 || cost < best) best = cost, *which = i;
        }
    }
    return best * p.blocks;
}

int fp8_tiles(bool exact, bool e8, int which, const Fp8Params& p, hipStream_t st) {
    if (exact) return e8 ? exact_of<true>(which, p, st) : exact_of<false>(which, p, st);
    return e8 ? tiles_of<Half, true>(which, p, st) : tiles_of<Half, false>(which, p, st);
}

}  // namespace tt
