"""GPU: products in 8-bit integers at the remainders of their tiles, in every form of D."""
import pytest
import torch

from tests.test_gpu_gemm_i8 import Case, FORMS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K", [(70, 1024, 300), (16, 7360, 200), (97, 259, 129)])
@pytest.mark.parametrize("d", [torch.float32, torch.bfloat16])
def test_added_by_tiles_of_32_rows(M, N, K, d):
    """Old values are a tile's own: what neighbouring tiles write meanwhile plays no part, however often the product is added."""
    c = Case(M, N, K, d, add=True, seed=K)
    c.run().check()
    for _ in range(20):
        c.old.copy_(c.d)
        c.run().check()
