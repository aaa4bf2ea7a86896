// Which tile a matrix product of tp_tile.hh takes, and how its contraction is split.
#include "tp_tile_plan.hh"

#include <algorithm>

#include "../../../include/torch_projectors_hip.h"

namespace tp {
namespace {

// One step (bk of the contraction) of a tile, and its start and end: among as many as a CU holds, and alone.  Measured on products of
// 1024 to 16384 along the contraction with every CU at work.
struct TileKind {
    int bm, bn, bk;
    double step_us, over_us, alone_us, alone_over_us;
};
constexpr TileKind kTiles16[] = {{64, 64, 64, 0.174, 2.2, 0.50, 5}, {128, 128, 64, 0.395, 5, 0.75, 6}, {256, 256, 64, 1.62, 10, 1.62, 10}};
constexpr TileKind kTilesStaged[] = {{64, 64, 64, 0.24, 1.4, 0.75, 5}, {128, 128, 64, 0.48, 5, 0.85, 6}};
constexpr TileKind kTiles32[] = {{64, 64, 32, 0.44, 0.5, 0.62, 4}, {128, 128, 32, 1.42, 3, 1.42, 4}, {256, 128, 32, 2.40, 11, 2.40, 11}};
const TileKind& kind_of(int dt, const TilePlan& t) {
    return dt == TP_F32 ? kTiles32[t.tile] : t.direct ? kTiles16[t.tile] : kTilesStaged[t.tile];
}
constexpr int kMaxSplits = 32;

}  // namespace

// The tile, and the tiles and ranges that are split, with the least time by a count of steps.  Every CU computes as many whole
// tiles; those that are left over are split along the contraction so that they give every CU something to do, too, which
// costs their sums written and read (by one workgroup a tile, at some 70 GB/s).  Against all tiles and 1 to 16 ranges
// on 56 products from 20 x 5000 to 4096 x 12288 the choice is 2.1 % from the best on average, at most 21 %.
TilePlan tile_plan(int dt, bool direct, int64_t rows, int64_t cols, int64_t kdim) {
    const int kinds = dt == TP_F32 || direct ? 3 : 2;
    TilePlan best{direct, kinds - 1, 0, 1};  // (the fewest tiles: where these are more than a launch holds the product refuses)
    double least = 1e300;
    for (int t = 0; t < kinds; ++t) {
        const TileKind& k = kind_of(dt, TilePlan{direct, t, 0, 1});
        const int64_t tiles = ((rows + k.bm - 1) / k.bm) * ((cols + k.bn - 1) / k.bn);
        if (tiles > kMaxTiles) continue;
        const int64_t steps = (kdim + k.bk - 1) / k.bk;
        auto weigh = [&](int64_t each, int s) {  // `each` whole tiles on a CU, the others in s ranges
            const int64_t rest = tiles - each * kCus, groups = (rest * s + kCus - 1) / kCus, part = (steps + s - 1) / s;
            double us = each * (steps * k.step_us + k.over_us) + groups * (part * k.step_us + k.over_us);
            us = std::max(us, (each ? steps : part) * k.alone_us + k.alone_over_us);
            if (s > 1) us += 6.0 + 0.1 * s + (s + 1) * (k.bm * k.bn * 6e-5) * double((rest + kCus - 1) / kCus);
            if (us < least) {
                least = us;
                best = {direct, t, uint32_t(each * kCus), s};
            }
        };
        weigh(tiles / kCus, 1);
        for (int s = 2; s <= kMaxSplits && s <= steps; ++s) {
            if (tiles % kCus) weigh(tiles / kCus, s);
            if (tiles >= kCus && tiles * s <= 8 * kCus) weigh(0, s);
        }
    }
    return best;
}
int64_t tile_part_bytes(int dt, const TilePlan& t, int64_t rows, int64_t cols) {
    const TileKind& k = kind_of(dt, t);
    const int64_t rest = tile_count(dt, t, rows, true) * tile_count(dt, t, cols, false) - int64_t(t.whole);
    return t.splits > 1 && rest > 0 ? rest * t.splits * k.bm * k.bn * 4 : 0;
}
int64_t tile_count(int dt, const TilePlan& t, int64_t n, bool of_rows) {
    const int size = of_rows ? kind_of(dt, t).bm : kind_of(dt, t).bn;
    return (n + size - 1) / size;
}

}  // namespace tp
