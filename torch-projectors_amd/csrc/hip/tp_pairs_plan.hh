// How a call of the pair log probabilities is cut into workgroups, ranges and pieces: sizes alone, on the host.
#pragma once

#include <stdint.h>

#include "../../../include/torch_projectors_hip.h"
#include "tp_tile_plan.hh"

namespace tp {

constexpr int64_t kMaxPairRows = int64_t(1) << 26;  // of either side
constexpr int64_t kMaxPairs = int64_t(1) << 35;     // images times references: fewer than kMaxTiles tiles of 128 x 128 on both sides
constexpr int kFewImages = 8;                       // up to here the references are streamed past the images

constexpr int kFewWaves = 8, kAhead = 4, kUnit = 128;  // of k_pairs_few
constexpr int kBackCols = 4, kBackRows = 64;           // of k_pairs_few_back

inline int64_t up_to(int64_t n, int64_t multiple) { return (n + multiple - 1) / multiple * multiple; }
inline int64_t up16(int64_t bytes) { return up_to(bytes, 16); }
inline int size_of(int dt) { return dt == TP_F32 ? 4 : 2; }

// ------------------------------------------------------------------ few images
// Ranges of the rows' values: as many workgroups as hide a load's way, each of at least a round of loads, and 16 at most, as one workgroup an image
// adds them up (1 x 16 x 262144 bfloat16 26 us, in 128 ranges 42; 1 x 40 x 16640 float32 13.1, in 17 ranges 13.9).
inline int few_splits(int dt, int64_t N, int64_t K) {
    const int64_t groups = (N + 15) / 16, units = (K * size_of(dt) + kUnit - 1) / kUnit;
    int64_t s = (2 * kCus + groups - 1) / groups;
    const int64_t most = (units + kFewWaves * kAhead - 1) / (kFewWaves * kAhead);
    if (s > most) s = most;
    return int(s < 1 ? 1 : s > 16 ? 16 : s);
}
// References that a workgroup joins: all of them up to 8192, which it reads in two steps, and a step's each beyond, whose parts take a
// launch more (1 x 36864 x 1024 bfloat16 24 us, in one workgroup 5 us longer).
inline int64_t few_each(int64_t N) { return N <= 8192 ? N : 4096; }
inline int64_t few_parts(int64_t N) { return (N + few_each(N) - 1) / few_each(N); }
// References of a range of the gradient.
inline int64_t few_per(int64_t N, int64_t K) {
    const int64_t blocks = (K + 256 * kBackCols - 1) / (256 * kBackCols);
    int64_t ranges = (4 * kCus + blocks - 1) / blocks;
    int64_t per = (N + ranges - 1) / ranges;
    per = up_to(per, 8);
    return per < 16 ? 16 : per;
}

// ------------------------------------------------------------------ many images: the gradient
// The scores' gradient G is formed for a piece of the references and one of the images at a time.  A piece of G is at most
// kPieceBytes large (128 MB stay in the last cache between the product that writes it and those that read it), and of at
// most kPieceImages images: their rows' distance is within what the products' 32-bit offsets reach, and G's 256 references at least within its bytes
// (1048576 x 512 x 1024 float32 25 ms a step, in pieces of all images 30).  16-bit rows are multiplied with G in two pieces of their type, what the first leaves to the second: four bytes of G either way.
constexpr int64_t kPieceBytes = int64_t(1) << 27, kPieceImages = int64_t(1) << 15;

inline int g_pieces(int dt) { return dt == TP_F32 ? 1 : 2; }

struct BackLayout {
    int64_t images, references;  // of a piece, at most
    int64_t ldg;                 // elements of a row of G (a reference's) or, of 16 bits, of each of its two pieces, the second behind the first
    TilePlan grad, refs, imgs;   // G, the references' gradient, the images'
    // bytes from the workspace's start: coefficients, scale and flag, G, its sums over the images, the split tiles' sums, and sums over
    // the pieces of the images (of a piece's references) and of the references (of all images)
    int64_t coef, scale, g, sums, part, dr, dx, bytes;
};
// n in equal parts of at most `most` (a multiple of 256), whole multiples of 256 where there are several
inline int64_t equal_parts(int64_t n, int64_t most) {
    const int64_t parts = (n + most - 1) / most, each = up_to((n + parts - 1) / parts, 256);
    return each < n ? each : n;
}
inline BackLayout back_layout(int dt, bool direct, int64_t M, int64_t N, int64_t K, bool d_x, bool d_r) {
    BackLayout b{};
    b.images = equal_parts(M, kPieceImages);
    b.ldg = up_to(b.images, 8);
    int64_t most = kPieceBytes / (b.ldg * 4) / 256 * 256;
    // (a piece's gradients are at most kMaxTiles tiles of 128 x 128: 32768 references of the longest rows, and as many images)
    const int64_t fit = kMaxTiles / ((K + 127) / 128) * 128 / 256 * 256;
    if (most > fit) most = fit;
    if (most < 256) most = 256;
    b.references = equal_parts(N, most);
    b.grad = tile_plan(dt, direct, b.references, b.images, K);
    b.refs = tile_plan(dt, direct, b.references, K, g_pieces(dt) * b.images);
    b.imgs = tile_plan(dt, direct, b.images, K, g_pieces(dt) * b.references);
    int64_t at = 0;
    auto room = [&](int64_t bytes) {
        const int64_t here = at;
        at += up16(bytes);
        return here;
    };
    b.coef = room(M * 16);
    b.scale = room(16);
    b.g = room(b.references * b.ldg * 4);
    b.sums = room(tile_count(dt, b.grad, b.images, false) * b.references * 4);
    int64_t part = tile_part_bytes(dt, b.grad, b.references, b.images);
    auto also = [&](int64_t bytes) { part = part > bytes ? part : bytes; };
    if (d_r) also(tile_part_bytes(dt, b.refs, b.references, K));
    if (d_x) also(tile_part_bytes(dt, b.imgs, b.images, K));
    b.part = room(part);
    b.dr = room(d_r && b.images < M ? b.references * K * 4 : 0);
    b.dx = room(d_x && b.references < N ? M * K * 4 : 0);
    b.bytes = at;
    return b;
}

}  // namespace tp
