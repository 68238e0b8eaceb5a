// The gated half of a feed-forward block in 8 bits on workgroup tiles.
#include "tt_fp8_tiles.hpp"

namespace tt {

namespace {

template <typename T, bool E8>
int tiles_of(int which, const Fp8Params& p, hipStream_t st) {
    switch (which) {
        case 0:
            return tiles_run<T, E8, true, 2, 4, 8, 4, 2>(p, st);
        case 1:
            return tiles_run<T, E8, true, 2, 4, 4, 4, 3>(p, st);
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

double fp8_gated_tiles_cost(const Fp8Params& p, int kind, int* which) {
    const int shapes[5][2] = {{256, 128}, {128, 128}, {128, 64}, {64, 64}, {64, 32}};
    const double steps[5] = {1.38, 0.95, 0.52, 0.345, 0.225};
    const int code_shapes[4] = {256, 128, 64, 32};
    const double code_steps[4] = {1.38, 0.95, 0.65, 0.45};
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
        for (int i = 0; i < 5; ++i) {
            const double cost = tiles_cost(p, shapes[i][0], shapes[i][1], steps[i]);
            if (i == 0 || cost < best) best = cost, *which = i;
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

}  // namespace tt
