// Which kernel a product of packed tensors or a weight gradient from one (om_gemm8.hip) runs on: host code alone, by sizes and
// the number of CUs, so that a test can tell which kernels its sizes reach.
#pragma once

#include <cmath>

#include "om_internal.hpp"

namespace om8 {

// A kernel's tile and what its workgroups take, in us, with `resident` of them on a CU at most: `fix` a round of those and
// `each` a workgroup, and for a block of k `alone` where a CU has one workgroup, `shared` a workgroup where it has more; with
// every CU busy the clock falls and the caches fill, and a block takes `chip` a workgroup and CU. Fitted to 3402 (products) and
// 5844 (weight gradients) times over all kernels, splits of k and sizes from 1 to 16384; the choice by them is 0.8 % (0.3 %)
// behind the best of all those in the mean, 15 % (19 %) at most.
struct Tile {
    int bm, bn, resident;
    float fix, each, alone, shared, chip;
};
struct Choice {
    int tile, splits;
};
// Splitting k costs a second launch that adds the parts, `join` us and `join_each` a million values; `most` parts of `least` blocks
// (weight gradients of few columns gain from up to 32 parts of two: 16384 x 64 x 64 11.5 us, 12.8 by 16 of four; products do not).
template <int N>
Choice choose(const Tile (&tiles)[N], int cus, int64_t m, int64_t n, int blocks, int64_t row_bytes, float join, float join_each, int most,
              int least) {
    Choice best = {-1, 1};
    double shortest = 0.0;
    // comparisons of one kernel or split: a number that is none of them leaves no choice
    const char *only_tile = om::tuning_env("OM_TILE8"), *only_splits = om::tuning_env("OM_SPLITS8");
    for (int t = 0; t < N; t++) {
        const Tile &c = tiles[t];
        if (only_tile && atoi(only_tile) != t) continue;
        if ((c.bm > c.bn ? c.bm : c.bn) * row_bytes > INT64_C(0xFFFFFFFF)) continue;  // offsets inside a tile: 32 bits
        for (int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
            if (s > 1 && (s > most || blocks < least * s)) break;
            if (only_splits && atoi(only_splits) != s) continue;
            const int per = (blocks + s - 1) / s, parts = per ? (blocks + per - 1) / per : 1;
            const double wgs = (double)((m + c.bm - 1) / c.bm) * (double)((n + c.bn - 1) / c.bn) * parts;
            const double load = std::ceil(wgs / cus), rounds = std::ceil(load / c.resident);
            double us = c.fix * rounds + c.each * load +
                        std::fmax(std::fmax(c.alone * rounds, c.shared * load), c.chip * wgs / cus) * per;
            if (parts > 1) us += join + join_each * parts * (double)m * (double)n * 1e-6;
            if (best.tile < 0 || us < shortest) {
                shortest = us;
                best = {t, s};
            }
        }
    }
    return best;
}
// Blocks of k to a split and the splits that gives.
inline void split_blocks(int blocks, int splits, int &per, int &parts) {
    per = (blocks + splits - 1) / splits;
    parts = blocks > per ? (blocks + per - 1) / per : 1;
}

// k_gemm8<256, 256>, <128, 128>, <128, 64>, <64, 64>, k_gemm8_few<4>, <8>
constexpr Tile kTiles[] = {{256, 256, 1, 10.01f, 0.3f, 2.673f, 0.426f, 3.006f}, {128, 128, 2, 0.0f, 2.66f, 0.856f, 0.42f, 0.99f},
                           {128, 64, 3, 0.0f, 1.27f, 0.669f, 0.436f, 0.504f},   {64, 64, 4, 0.07f, 0.52f, 0.497f, 0.293f, 0.24f},
                           {32, 32, 4, 0.47f, 0.33f, 0.08f, 0.088f, 0.095f},    {32, 32, 2, 0.0f, 0.79f, 0.021f, 0.075f, 0.086f}};
inline Choice choose_product(int cus, int64_t m, int64_t n, int blocks, int64_t row_bytes) {
    return choose(kTiles, cus, m, n, blocks, row_bytes, 2.5f, 0.69f, 16, 4);
}

// k_gemm8_thin<NW, MR>: 16 MR rows by NW wavefronts, MR = 0 where the others are taken. Up to 48 rows it is the fastest (17 x 2048 x
// 2048 4.0 us, the best of the others 4.9; 40 x 2048 x 2048 4.6 and 5.0; 64 by such a kernel 5.3 and 5.0) until a wavefront has so
// many blocks one after the other that the others, or a split of k, are (16 x 64 x 12000 7.7 us and 6.6, 32 x 256 x 8192 7.3 and
// 6.9, 40 x 512 x 6000 6.9 and 6.8).
struct Thin {
    int mr, nw;
    int64_t groups;
};
inline Thin choose_thin(int cus, int64_t m, int64_t n, int blocks) {
    constexpr int kMostBlocks[] = {64, 48, 40};
    const int64_t mr = (m + 15) / 16, groups = (n + 15) / 16;
    if (mr > 3 || blocks > kMostBlocks[mr - 1]) return Thin{0, 0, 0};
    return Thin{(int)mr, groups <= cus ? 8 : 4, groups};
}

// k_dw8<4, 2>, <2, 2>, <1, 3>, k_dw8_few<8>
constexpr Tile kTilesDw[] = {{32, 128, 2, 0.71f, 1.75f, 0.794f, 0.696f, 0.663f},
                             {32, 64, 3, 0.83f, 0.65f, 0.525f, 0.429f, 0.456f},
                             {32, 32, 2, 0.0f, 0.61f, 0.523f, 0.38f, 0.375f},
                             {32, 32, 1, 0.3f, 0.55f, 0.31f, 0.314f, 0.348f}};
inline Choice choose_dw(int cus, int64_t m, int64_t n, int blocks, int64_t row_bytes) {
    return choose(kTilesDw, cus, m, n, blocks, row_bytes, 2.14f, 0.92f, 32, 2);
}

}  // namespace om8
