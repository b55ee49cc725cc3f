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


class Placed(Case):
    """A case whose D begins `shift` elements behind a 16-byte boundary, in rows of ldd."""

    def __init__(self, M, N, K, d, bias, add, ldd, shift, seed):
        super().__init__(M, N, K, d, bias, add, seed=seed)
        old = self.d[:M, :N].clone()
        self.ldd = ldd
        self.whole = torch.full((shift + (M + 1) * ldd + 8,), -5.0, device="cuda", dtype=d)
        self.shift, self.d = shift, self.whole[shift:shift + (M + 1) * ldd].view(M + 1, ldd)
        self.d[:M, :N] = old
        self.old = self.d.clone()

    def check(self):
        super().check()
        n = self.shift + self.d.numel()
        assert bool((self.whole[:self.shift] == -5).all()) and bool((self.whole[n:] == -5).all())


# all of these have more tiles than there are SMs, whatever the tiles: they are computed by pairs of CTAs
@pytest.mark.parametrize("d,bias,add", FORMS)
@pytest.mark.parametrize("M,N,K", [(4111, 4104, 300), (2049, 7368, 129), (4100, 4112, 1024), (2300, 9000, 16)])
def test_pairs_whose_rows_are_whole_16_bytes(M, N, K, d, bias, add):
    """Results by tensor-map copies: widths that are multiples of 8 and not of 32, odd numbers of rows; strips that do not exist beside strips that are added."""
    Case(M, N, K, d, bias, add, seed=N).run().check()
    Placed(M, N, K, d, bias, add, N + 24, 0, seed=N).run().check()       # what is between the rows stays


@pytest.mark.parametrize("d,bias,add", FORMS)
@pytest.mark.parametrize("N,ldd,shift", [(4104, 4104, 1), (4104, 4104, 2), (4104, 4105, 0), (4102, 4112, 0), (4101, 4104, 3)])
def test_pairs_whose_rows_are_not(N, ldd, shift, d, bias, add):
    """A base, a pitch or a width that is no whole 16 bytes, each alone: results one by one."""
    Placed(4111, N, 300, d, bias, add, ldd, shift, seed=shift).run().check()


@pytest.mark.parametrize("d,bias,add", FORMS)
def test_few_rows_and_columns_of_many(d, bias, add):
    """Tall and wide products, which fit into one round of tiles or not."""
    for M, N, K in ((40000, 8, 64), (20000, 40, 513), (8, 40000, 64), (40, 40000, 513), (33, 19000, 1024)):
        Case(M, N, K, d, bias, add, seed=M).run().check()
