// Which tile a matrix product of tp_tile.hh takes (tp_tile_plan.hip).
#pragma once

#include <stdint.h>

namespace tp {

constexpr int kCus = 256;
constexpr int64_t kMaxStride = int64_t(1) << 21;  // elements between an operand's rows, and values of a row
constexpr int64_t kMaxTiles = int64_t(1) << 22;  // of a product (a launch has fewer than 2^32 lanes)

struct TilePlan {
    bool direct;     // operands go straight to LDS (16-bit rows that start at 16-byte boundaries)
    int tile;        // 0: 64 x 64, 1: 128 x 128, 2: 256 x 256 (float32: 256 x 128)
    uint32_t whole;  // tiles that are not split
    int splits;      // ranges of the contraction of the others
};
// rows, columns and contraction of a product of a type -> its tile and ranges
TilePlan tile_plan(int dt, bool direct, int64_t rows, int64_t cols, int64_t kdim);
// bytes that the split tiles' sums need
int64_t tile_part_bytes(int dt, const TilePlan& t, int64_t rows, int64_t cols);
int64_t tile_count(int dt, const TilePlan& t, int64_t n, bool of_rows);  // along the rows or the columns

}  // namespace tp
