"""Register, scratch and LDS budgets of the tiled products and their companions (CPU: the compiler's report beside the objects,
or a fresh compile when it is stale)."""
import pytest

from tests.test_kernel_resources_cpu import GRANULE, LDS_PER_CU, _kernels, _report

SOURCES = ("tp_pairs.hip", "tp_pairs_f32.hip", "tp_pairs_f16.hip", "tp_pairs_bf16.hip", "tp_rows8.hip")


@pytest.fixture(scope="module")
def kernels():
    return {src: _kernels(_report(src), "k_") for src in SOURCES}


@pytest.mark.parametrize("src", SOURCES)
def test_no_kernel_spills(kernels, src):
    assert kernels[src], "no kernels in the resource report"
    bad = {n: k["ScratchSize"] for n, k in kernels[src].items() if k["ScratchSize"]}
    assert not bad, bad


@pytest.mark.parametrize("src,tile,per_cu", [
    ("tp_pairs_bf16.hip", "Li64ELi64E", 4), ("tp_pairs_bf16.hip", "Li128ELi128E", 2), ("tp_pairs_bf16.hip", "Li256ELi256E", 1),
    ("tp_pairs_f16.hip", "Li64ELi64E", 4), ("tp_pairs_f16.hip", "Li128ELi128E", 2), ("tp_rows8.hip", "Li64ELi64E", 4),
    ("tp_rows8.hip", "Li128ELi128E", 2), ("tp_pairs_f32.hip", "Li64ELi64E", 3), ("tp_pairs_f32.hip", "Li128ELi128E", 1),
    ("tp_pairs_f32.hip", "Li256ELi128E", 1)])
def test_tiles_fit_the_lds(kernels, src, tile, per_cu):
    """What the tiles' plan counts on a CU's holding."""
    hits = [k for n, k in kernels[src].items() if "6k_tileI" in n and "TileShapeI" + tile in n]
    assert hits
    for k in hits:
        assert -(-k["LDS"] // GRANULE) * GRANULE * per_cu <= LDS_PER_CU, k


@pytest.mark.parametrize("src", ["tp_pairs_bf16.hip", "tp_pairs_f16.hip", "tp_rows8.hip"])
def test_registers_leave_two_middle_tiles_a_cu(kernels, src):
    """Operands that go straight to LDS: two workgroups of 8 wavefronts, four wavefronts a SIMD."""
    hits = [k for n, k in kernels[src].items() if "6k_tileI" in n and "Li128ELi128ELi2ELi4ELb0EEELb" in n and "ELb1ENS_" in n]
    assert hits and all(k["Occupancy"] >= 4 for k in hits), hits
