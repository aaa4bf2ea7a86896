"""What the kernels of the pair log probabilities take from their plans on trust holds for every size that calls accept: strides
and extents that 32-bit offsets reach, tiles that a launch holds, a workspace that is enough.  On the CPU."""
import math
import random

import pytest

from tests import pairs_plans as P
from torch_projectors import capi

SIZES = {P.F32: 4, P.F16: 2, P.BF16: 2}


def accepted(rng):
    """A call's sizes: rows of either side up to 2^26, 2^35 pairs, rows of up to 2^21 values."""
    def log(a, b):
        return int(math.exp(rng.uniform(math.log(a), math.log(b))))

    M = rng.choice([log(9, 1 << 26), log(9, 1 << 14)])
    N = rng.choice([log(1, 1 << 26), log(1, 4096)])
    N = max(1, min(N, P.limit(2) // M))
    return M, N, rng.choice([log(1, 1 << 21), 8 * log(1, 1 << 18), log(1, 20000)])


ENDS = [(1 << 26, 512, 8), (1 << 26, 512, 1 << 21), (9, 1 << 26, 1 << 21), (9, 1 << 26, 1), (512, 1 << 26, 64), (1 << 22, 8192, 16385), (5000000, 256, 2048),
        (5000000, 1024, 1024), (9000000, 512, 4224), (32769, 1 << 20, 8), (32768, 1 << 20, 1 << 21), (185363, 185363, 1 << 21), (129, 1 << 26, 129)]


def check(dt, M, N, K):
    for direct in ([True, False] if dt != P.F32 and K % 8 == 0 else [False]):
        where = (dt, direct, M, N, K)
        b = P.back_layout(dt, direct, M, N, K)
        assert 1 <= b.images <= M and 1 <= b.references <= N, where
        pieces = -(-M // b.images) * -(-N // b.references)
        assert pieces <= 1 << 22, where  # (a loop on the host)
        # rows of G as an operand: a tile's 256 rows of either side, or a step's 64, from one base
        row = b.ldg * 4  # (of 16 bits in two pieces)
        assert 2 * b.ldg <= P.limit(1) and 256 * row + row <= 0x7fffffff, where
        assert b.g_bytes <= 1 << 27, where
        for tile in (b.grad, b.refs, b.imgs, P.tile_plan(dt, direct, N, M, K)):
            assert 1 <= tile.tiles <= P.limit(0), where
            assert tile.whole <= tile.tiles and 1 <= tile.splits <= 32, where
        need = capi.lib().tp_pair_log_probs_back_work(dt, M, N, K, 1, 1)
        assert need >= b.bytes > 0, where


@pytest.mark.parametrize("dt", [P.F32, P.F16, P.BF16])
def test_every_accepted_size_fits_the_kernels(dt):
    for M, N, K in ENDS:
        check(dt, M, N, K)
    rng = random.Random(7 + dt)
    for _ in range(1500):
        check(dt, *accepted(rng))


@pytest.mark.parametrize("dt", [P.F32, P.F16, P.BF16])
def test_rows_of_inputs_that_offsets_reach(dt):
    """256 rows as far apart as is taken, and a row's values."""
    stride = P.limit(1)
    extent = (255 * stride + stride) * SIZES[dt]
    assert extent <= (1 << 32) - 1 if dt == P.F32 else extent <= 0x7fffffff


def test_tiles_of_integer_scores():
    """2^26 rows of either side and 2^37 scores at most."""
    rng = random.Random(1)
    for _ in range(3000):
        M = int(math.exp(rng.uniform(0, math.log(1 << 26))))
        N = max(1, min(int(math.exp(rng.uniform(0, math.log(1 << 26)))), (1 << 37) // M))
        K = 64 * rng.randint(1, 1024)
        t = P.tile_plan(P.BF16, True, M, N, K)
        assert 1 <= t.tiles <= P.limit(0), (M, N, K)


def test_small_calls_are_in_one_piece():
    for dt, M, N in ((P.BF16, 4096, 4096), (P.F32, 2048, 8192), (P.F16, 333, 1999)):
        b = P.back_layout(dt, True if dt != P.F32 else False, M, N, 4224)
        assert (b.images, b.references) == (M, N)


def forms(sizes, dt):
    """(product, tile, straight to LDS, in ranges) that calls of these sizes run."""
    out = set()
    for M, N, K in sizes:
        direct = dt != P.F32 and K % 8 == 0
        b = P.back_layout(dt, direct, M, N, K)
        for name, t in (("grad", b.grad), ("references", b.refs), ("images", b.imgs), ("scores", P.tile_plan(dt, direct, N, M, K))):
            out.add((name, t.tile, direct, t.split))
    return out


@pytest.mark.parametrize("dt", [P.F16, P.BF16])
def test_sizes_of_the_rounding_tests_reach_every_tile(dt):
    from tests.test_gpu_pairs_rounding import ROUNDED
    ran = forms(ROUNDED, dt)
    for name in ("references", "images"):
        for tile, direct in ((0, True), (1, True), (2, True), (0, False), (1, False)):
            assert any(f[:3] == (name, tile, direct) for f in ran), (name, tile, direct)
        assert any(f[0] == name and f[2] and f[3] for f in ran) and any(f[0] == name and not f[2] and f[3] for f in ran), name


def test_sizes_of_the_long_sums_reach_both_tiles_with_two_sums():
    from tests.test_gpu_pairs_float32 import LONG_SUMS
    ran = forms(LONG_SUMS, P.F32)
    for name in ("images", "references"):
        assert {f[1] for f in ran if f[0] == name} == {0, 1}, (name, ran)


def test_sizes_of_the_long_rows_reach_the_large_tiles_with_two_sums():
    from tests.test_gpu_pairs_float32 import LONG_ROWS
    ran = forms(LONG_ROWS, P.F32)
    assert {f[1:] for f in ran if f[0] == "scores"} == {(1, False, True), (2, False, False), (2, False, True)}


def test_sizes_of_the_masked_tests_reach_the_largest_tiles():
    from tests.test_gpu_pairs_masked_tiles import LARGE, MASKED
    for dtype, M, N, K in MASKED:
        dt = P.CODES[str(dtype)]
        b = P.back_layout(dt, dt != P.F32, M, N, K)
        assert b.imgs.tile == 2 and (b.references < N or N == 100), (dtype, M, N, K)
    for dtype, M, N, K in LARGE:
        dt = P.CODES[str(dtype)]
        assert P.tile_plan(dt, dt != P.F32, N, M, K).tile == 2, (dtype, M, N, K)


def test_ranges_of_few_images():
    """16 at most, and none without a round of loads."""
    rng = random.Random(3)
    for _ in range(2000):
        dt = rng.choice([P.F32, P.F16, P.BF16])
        N, K = int(math.exp(rng.uniform(0, 14))), int(math.exp(rng.uniform(0, math.log(1 << 21))))
        s = P.lib().splits(dt, P._L(N), P._L(K))
        units = -(-K * SIZES[dt] // 128)
        assert 1 <= s <= 16 and (s == 1 or s <= -(-units // 32)), (dt, N, K, s)


def test_more_tiles_than_a_launch_holds():
    """No call is accepted that has them; the plan is the one of the fewest tiles, and the product refuses."""
    for dt, direct, tile in ((P.F16, False, 1), (P.BF16, True, 2), (P.F32, False, 2)):
        t = P.tile_plan(dt, direct, 1 << 26, 1 << 21, 64)
        assert t.tile == tile and t.tiles > P.limit(0)


def test_no_kernels_that_no_call_reaches():
    """Codes go straight to LDS: no tiles that are staged in registers."""
    from tests.test_kernel_resources_cpu import _kernels, _report
    tiles = [n for n in _kernels(_report("tp_rows8.hip"), "k_") if "6k_tileI" in n]
    assert len(tiles) == 6 and all("ELb0ELb0ELb1ENS" in n for n in tiles), tiles
