// Which kernel and tile a gated product takes: the rules alone, on the host.
#pragma once

#include "gemm_choice.hpp"

namespace cuvit::detail {

/// The ring kernel's tiles, rows x outputs (of 2 n columns: twice as many B rows).
enum class GatedTile { k64x32Alone, k64x64, k64x64Alone, k128x64, k192x128, k256x128, k320x128 };
enum class GatedTileF32 { k32x16Alone, k32x32, k32x32Alone, k64x32 };

/// Rows that the kernel for few rows takes at most, four MFMA tiles of 16 (half as
/// many of operands that the ring takes too).
constexpr int kGatedRows = 64;

/// The product with 2 n columns whose tile grid the gated one's is.
inline GemmArgs gated_grid(const GatedArgs& args) {
    GemmArgs grid{};
    grid.m = args.m;
    grid.n = 2 * args.n;
    grid.k = args.k;
    grid.transposed = true;
    grid.count = 1;
    return grid;
}

struct GatedChoice {
    GatedTile tile;
    gemm::TileMap map;
};

/// The bf16 tile with the least cost: a CU's turns, each a tile's time, in us
/// fixed + by_k K. Fitted to MI355X times of (n, k) = (512, 192), (1024, 384),
/// (1365, 512), (2048, 768) and (1900, 1096) on 17 to 12608 rows, less 2.5 us of a
/// launch; the tile taken is the fastest or within a tenth of it in nearly all. Of
/// 2048 x 768, in us:
///   rows      64x32 alone  64x64   128x64  192x128  256x128  320x128
///   197           5.5        6.5      8.6     15.5     18.7     22.1
///   788          13.4       10.7     11.2     17.1     20.3     23.3
///   1576         21.9       19.9     14.7     17.8     21.4     24.8
///   3152         35.5       29.5     25.6     33.2     23.1     25.8
///   4616         50.9       38.8     35.6     34.9     42.1     30.4
///   12608       132        103       87.6     87.7     85.8     80.8
/// A tile that is the only one of its CU has nothing beside it to cover its waits:
/// up to 64 outputs it costs half as much again, with three stages a quarter
/// (394 rows: 9.2 -> 7.2 us), and below one such tile of 32 outputs a CU,
/// loading wavefronts beside the computing ones are the fastest.
inline GatedChoice choose_gated(const GatedArgs& args, int units) {
    struct Candidate {
        GatedTile tile;
        int rows;
        int outputs;
        double fixed;
        double by_k;
        double alone;
    };
    constexpr Candidate kCandidates[] = {
        {GatedTile::k64x64, 64, 64, 0.8, 0.0041, 1.25},    {GatedTile::k128x64, 128, 64, 1.3, 0.0066, 1.5},
        {GatedTile::k192x128, 192, 128, 3.5, 0.0165, 1.0}, {GatedTile::k256x128, 256, 128, 4.4, 0.0209, 1.0},
        {GatedTile::k320x128, 320, 128, 6.0, 0.0243, 1.0},
    };
    const GemmArgs grid = gated_grid(args);
    if (tile_count(grid, 64, 64) <= units) {
        return {GatedTile::k64x32Alone, tile_map(grid, 64, 64, 2)};
    }
    const int slots = units >= kXcds ? units / kXcds : 1; // CUs of an XCD
    GatedChoice best{};
    double best_cost = 0.0;
    for (const Candidate& c : kCandidates) {
        const int columns = 2 * c.outputs;
        int rounds = 0;
        gemm::TileMap map = balanced_map(grid, c.rows, columns, slots, &rounds);
        if (map.px == 0) { // too few tiles for a block to each XCD: in row-major order
            rounds = static_cast<int>((largest_share(grid, map, c.rows, columns) + slots - 1) / slots);
        }
        const double cost = rounds * (c.fixed + c.by_k * args.k) * (rounds == 1 ? c.alone : 1.0);
        if (best_cost == 0.0 || cost < best_cost) {
            best_cost = cost;
            best = {rounds == 1 && c.tile == GatedTile::k64x64 ? GatedTile::k64x64Alone : c.tile, map};
        }
    }
    return best;
}

/// The fp32 tile: these are bound by the MFMAs (137 TFLOP/s, what the clock under
/// them allows, on 6304 x 2048 x 768), so what counts is how evenly the tiles fall
/// on the CUs: 64 x 32 outputs against 32 x 32, a tile's time 1.9 to 1 (788 rows of
/// 2048 x 768: 49.1 and 47.1 us; 6304: 289 and 302).
inline GatedTileF32 choose_gated_f32(const GatedArgs& args, int units) {
    const GemmArgs grid = gated_grid(args);
    if (tile_count(grid, 32, 32) <= units) {
        return GatedTileF32::k32x16Alone;
    }
    const std::int64_t small = (tile_count(grid, 32, 64) + units - 1) / units;
    const std::int64_t large = (tile_count(grid, 64, 64) + units - 1) / units;
    if (small == 1) {
        return GatedTileF32::k32x32Alone;
    }
    const double large_cost = large == 1 ? 2.9 : 1.9 * static_cast<double>(large);
    return large_cost < static_cast<double>(small) ? GatedTileF32::k64x32 : GatedTileF32::k32x32;
}

/// The fp32 XCD split: none where the columns of tiles are a multiple of the XCDs,
/// since tiles in row-major order then give each XCD columns of its own (6304 x 2048
/// x 768: 293 us so, 305 in blocks); else balanced_map's blocks, without which every
/// XCD reads all of B (2308 x 1365 x 512: 147 MB fetched, 65 -> 59 us).
inline gemm::TileMap gated_map_f32(const GatedArgs& args, int bm, int bn, int units) {
    const GemmArgs grid = gated_grid(args);
    int rounds = 0;
    return (grid.n + bn - 1) / bn % kXcds == 0 ? gemm::TileMap{0, 0}
                                               : balanced_map(grid, bm, bn, units >= kXcds ? units / kXcds : 1, &rounds);
}

} // namespace cuvit::detail
