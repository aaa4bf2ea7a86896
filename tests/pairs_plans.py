"""The plans of the tiled products and of the pair log probabilities' gradient (sizes alone, tp_tile_plan.hip and
tp_pairs_plan.hh), compiled for the host and called from tests that say which tile, form, ranges and pieces they mean to run."""
import ctypes
import functools
import os
import shutil
import subprocess
import tempfile
from typing import NamedTuple

import pytest

HIP = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torch-projectors_amd", "csrc", "hip")
F32, F16, BF16 = 0, 3, 4
CODES = {"torch.float32": F32, "torch.float16": F16, "torch.bfloat16": BF16}

SOURCE = """
#include "tp_tile_plan.hip"
#include "tp_pairs_plan.hh"
using namespace tp;
static void put(long long* o, const TilePlan& t, int dt, int64_t rows, int64_t cols) {
    o[0] = t.tile; o[1] = t.direct; o[2] = t.whole; o[3] = t.splits;
    o[4] = tile_count(dt, t, rows, true) * tile_count(dt, t, cols, false);
}
extern "C" void tile(int dt, int direct, long long rows, long long cols, long long kdim, long long* o) {
    put(o, tile_plan(dt, direct, rows, cols, kdim), dt, rows, cols);
}
extern "C" void back(int dt, int direct, long long M, long long N, long long K, int dx, int dr, long long* o) {
    const BackLayout b = back_layout(dt, direct, M, N, K, dx, dr);
    o[0] = b.images; o[1] = b.references; o[2] = b.ldg; o[3] = b.bytes; o[4] = b.sums - b.g;
    put(o + 5, b.grad, dt, b.references, b.images);
    put(o + 10, b.refs, dt, b.references, K);
    put(o + 15, b.imgs, dt, b.images, K);
}
extern "C" int splits(int dt, long long N, long long K) { return few_splits(dt, N, K); }
extern "C" long long limit(int which) { return which == 0 ? kMaxTiles : which == 1 ? kMaxStride : which == 2 ? kMaxPairs : kMaxPairRows; }
"""


class Tile(NamedTuple):
    tile: int    # 0: 64 x 64, 1: 128 x 128, 2: 256 x 256 (float32: 256 x 128)
    direct: int  # straight to LDS
    whole: int   # tiles that are not split
    splits: int  # ranges of the others
    tiles: int

    @property
    def split(self):
        return self.splits > 1 and self.tiles > self.whole


class Back(NamedTuple):
    images: int      # of a piece
    references: int
    ldg: int
    bytes: int
    g_bytes: int
    grad: Tile
    refs: Tile
    imgs: Tile


@functools.lru_cache(None)
def lib():
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("no host compiler")
    with tempfile.TemporaryDirectory() as d:
        src, so = os.path.join(d, "plans.cpp"), os.path.join(d, "plans.so")
        with open(src, "w") as f:
            f.write(SOURCE)
        subprocess.run([gxx, "-std=c++17", "-O1", "-shared", "-fPIC", "-I", HIP, src, "-o", so], check=True)
        return ctypes.CDLL(so)


_L = ctypes.c_longlong


def tile_plan(dt, direct, rows, cols, kdim):
    o = (_L * 5)()
    lib().tile(dt, int(direct), _L(rows), _L(cols), _L(kdim), o)
    return Tile(*o)


def back_layout(dt, direct, M, N, K, d_x=True, d_r=True):
    o = (_L * 20)()
    lib().back(dt, int(direct), _L(M), _L(N), _L(K), int(d_x), int(d_r), o)
    return Back(*o[:5], Tile(*o[5:10]), Tile(*o[10:15]), Tile(*o[15:20]))


def limit(which):
    lib().limit.restype = _L
    return lib().limit(which)
