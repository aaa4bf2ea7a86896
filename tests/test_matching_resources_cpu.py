"""Register, scratch and LDS budgets of the matching kernels (CPU: the compiler's report beside the objects, or a
fresh compile when it is stale): none spills, and what the rules for splitting work count on a CU's holding fits
there."""
import pytest

from tests.test_kernel_resources_cpu import GRANULE, LDS_PER_CU, _kernels, _report

SOURCES = ("tp_scores.hip", "tp_probs.hip", "tp_route.hip")


@pytest.fixture(scope="module")
def kernels():
    return {src: _kernels(_report(src), "k_") for src in SOURCES}


@pytest.mark.parametrize("src", SOURCES)
def test_no_kernel_spills(kernels, src):
    assert kernels[src], "no kernels in the resource report"
    bad = {n: k["ScratchSize"] for n, k in kernels[src].items() if k["ScratchSize"]}
    assert not bad, bad


@pytest.mark.parametrize("tile,per_cu", [("ILi64ELi64E", 4), ("ILi128ELi128E", 2), ("ILi256ELi256E", 1)])
def test_tiles_fit_the_lds(kernels, tile, per_cu):
    hits = [k for n, k in kernels["tp_scores.hip"].items() if "k_scores_tile" + tile in n]
    assert len(hits) == 2  # one per type of the scores
    for k in hits:
        assert -(-k["LDS"] // GRANULE) * GRANULE * per_cu <= LDS_PER_CU, k


def test_two_workgroups_of_log_probabilities_per_cu(kernels):
    hits = [k for n, k in kernels["tp_probs.hip"].items() if "7k_probsI" in n]
    assert len(hits) == 12  # 3 types of the scores, 1, 2, 4 or 8 wavefronts a row
    for k in hits:
        # 512 lanes: two wavefronts per SIMD each
        assert k["Occupancy"] >= 4 and 2 * -(-k["LDS"] // GRANULE) * GRANULE <= LDS_PER_CU, k
