"""Every compiled kernel of the rows by class is one that their plan can choose (CPU, from the compiler's report)."""
import re

from tests.test_kernel_resources_cpu import _kernels, _report


def test_sixteen_wavefronts_are_compiled_with_the_weights_gradient_only():
    names = [n for n in _kernels(_report("tp_route.hip"), "k_") if "_rows" in n]
    kinds = [re.search(r"Li(\d+)ELi(\d+)ELb([01])E", n).groups() for n in names]
    assert kinds and {dot for w, _, dot in kinds if w == "16"} == {"1"}
    assert {dot for w, _, dot in kinds if w == "4"} == {dot for w, _, dot in kinds if w == "1"} == {"0", "1"}
