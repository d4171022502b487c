// linear8_shape.h -- where the kernels of linear8.hip read and which of them a call
// takes, as plain C++ (compiled for the host alone by the tests).  The figures are an
// MI355X's, 256 CUs; a part of one is told apart by its number of CUs.
#pragma once

#include <algorithm>
#include <cstdint>

namespace ember {

// Operands are read through buffers of this many bytes from a tile's first row on, no
// fewer than its rows have: 256 of at most 2^23.  A load's offset has a lane's share,
// its place in the tile, and one that all lanes have, the group of k.  The lane's is the
// one that is sure to be held against the buffer's size, so past the last group it lies
// past the buffer: such a load gives 0 and reads nothing.
constexpr unsigned kBufferBytes = 0x80000000u;
constexpr unsigned lane_offset(unsigned in_tile, bool there)
{
    return in_tile | (there ? 0u : kBufferBytes);
}

// Rows of a few-rows workgroup, in sixteens.
inline int few_rows(int64_t n)
{
    return n <= 16 ? 1 : n <= 32 ? 2 : n <= 48 ? 3 : 4;
}
// Its columns, in sixteens: each workgroup reads all of a's rows, so many where
// those are, but not so many that more than three eighths of the CUs are left without
// one (a gated layer's, which has twice as many rows of w: none).  16 x 4096 x 16384: 64
// columns 15.7 us, 16 19.4; 16 x 4096 x 4096: 14.4 and 7.1; 1 x 4096 x 16384: 14.6
// and 14.0.
inline int few_columns(int64_t n, int64_t m, bool gated, int cus)
{
    if (gated) return n > 32 && (m + 31) / 32 >= cus ? 2 : 1;
    const int64_t least = 5 * (int64_t)cus;
    return n <= 8 ? 1 : 8 * ((m + 63) / 64) >= least ? 4 : 8 * ((m + 31) / 32) >= least ? 2 : 1;
}
// A workgroup's waves.  Two, so that several share a CU and none waits for the last;
// four for 64 columns, of which a CU has one workgroup (37 x 4096 x 16384: 18.3 us, with
// two 19.1, 16 x 8192 x 16384: 27.6 and 35.8), and where a CU has no more than one of
// 16 columns and 16 rows and there is more than a group or two of k for each wave.
// With four and with two, one row: 4096 columns of k = 1024 3.4 and 3.3 us, of 1536 3.8
// and 4.3, of 4096 6.5 and 7.4, of 16384 17.3 and 23.1; 256 columns of k = 2560 4.1 and
// 4.6; but 4500 columns, of which some CUs have two, with eight rows of k = 2048 6.7 and
// 6.3, of 4096 10.2 and 9.6.
constexpr bool four_waves(int64_t m, int groups, int cus)
{
    return (m + 15) / 16 <= cus && groups > 8;
}

// What a call costs with each kernel, in us, fitted to measured times of 24 products
// (65 x 4096 x 4096 to 8192 x 8192 x 8192) and 18 gated layers with every kernel and
// 1 to 16 splits of k, and of 56 and 66 with 1 to 128 rows and 2730 to 50000 columns:
// the choice by it is within 10 % of the fastest for those, within 5 % for nearly all;
// over 69 others at random 0.9 % on average, 19 % at most.  Few rows: a launch, and
// what a CU's workgroups read (13 bytes a cycle); the largest workgroups, of which a CU
// has one (a gated layer's: two), in whole rounds with their ends.  Tiles: a launch, and
// for each round over the CUs the ends of a tile and its stages, whose time is one
// workgroup's latency with the chip nearly empty and throughput with it full; the sums'
// way to memory; and for sums that are added or gated in a launch of their own, that and
// its bytes.
enum Kernel { kFew, kSmallTiles, kMidTiles, kLargeTiles };
struct Choice {
    Kernel kernel;
    int splits, chunk;
};
constexpr int kMostSplits = 16;

inline Choice choose(int64_t n, int64_t m, int groups, bool gated, int cus)
{
    const auto over = [](int64_t a, int64_t b) { return (double)((a + b - 1) / b); };
    const double moved = 4.0 * (gated ? 2 : 1) * n * m / 5e6;  // us to write the sums once
    Choice best = {kFew, 1, groups};
    const int nt = few_rows(n), mb = few_columns(n, m, gated, cus);
    const double units = over(n, 16 * nt) * over(m, 16 * mb);
    const int blocks = (gated ? 2 : 1) * mb;  // of 16 rows of w
    double few_rounds = std::max(1.0, units / cus), few_ends = 0.07 * nt * blocks * blocks;
    if (blocks == 4) few_rounds = gated ? 2 * over((int64_t)units, 2 * cus) : over((int64_t)units, cus);
    if (blocks == 4 && gated) few_ends = 0.5;
    double least = 2.2 + few_rounds * (few_ends + groups * 0.0656 * (nt + blocks)) + (gated ? 2.5 + moved : 0);
    const auto consider = [&](Kernel kernel, int splits, int chunk, double us) {
        if (us < least) least = us, best = {kernel, splits, chunk};
    };
    const auto rounds = [&](double tiles, double ends, double empty, double full) {
        return 3 + over((int64_t)tiles, cus) * (ends + groups * (empty + (full - empty) * std::min(1.0, tiles / cus)));
    };
    if (gated) {
        consider(kLargeTiles, 1, groups, rounds(over(n, 256) * over(m, 128), 9, 2.25, 3.05));
        consider(kMidTiles, 1, groups, rounds(over(n, 128) * over(m, 128), 8, 1.35, 1.7));
    } else {
        consider(kLargeTiles, 1, groups, rounds(over(n, 256) * over(m, 256), 6, 2.25, 2.95) + 0.5 * moved);
    }
    for (int want = 1; want <= kMostSplits; want *= 2) {
        const int chunk = want == 1 ? groups : ((groups + want - 1) / want + 3) / 4 * 4, splits = (groups + chunk - 1) / chunk;
        if (splits > 1 && splits * moved > 100) break;
        const double tiles = over(n, 128) * over((gated ? 2 : 1) * m, 128) * splits;
        double us = 6 + chunk * (tiles <= cus ? 0.81 + 0.23 * tiles / cus : over((int64_t)tiles, 2 * cus) * 1.77) + 0.5 * splits * moved;
        if (splits > 1 || gated) us += 3 + (splits + 1) * moved;
        consider(kSmallTiles, splits, chunk, us);
        if (splits < want) break;
    }
    return best;
}

// The same call where there is no memory for sums on their way: whole sums, which the
// kernel writes to the output itself.
inline Choice without_scratch(int groups, bool gated)
{
    return {gated ? kMidTiles : kSmallTiles, 1, groups};
}

}  // namespace ember
