"""Scores in 8-bit integers next to the sizes where another kernel takes them: by images, references and bytes of their codes."""
import pytest

from tests.test_gpu_rows8 import BF16, F32, m, scores  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("M,N,K", [(2, 16384, 128), (8, 16385, 128), (8, 16384, 300), (9, 8192, 128), (9, 8193, 128), (16, 8192, 1000), (16, 5041, 16640),
                                   (16, 5042, 16640), (17, 4096, 260), (32, 4097, 260), (32, 4096, 9216), (32, 4096, 9217), (33, 100, 260)])
def test_either_side_of_a_border(m, M, N, K, out):  # noqa: F811
    scores(m, M, N, K, out=out, seed=M + N)
