"""GPU: products in 8-bit integers of which single waits on the device run out while everything that they wait for is on its way.  Whichever of them do, the kernel ends
with its copies landed and its MMAs done, every result is the right one or NaN, nothing else is written, and the same product then runs as ever."""
import pytest
import torch

import lumi_b200
from tests.test_gpu_gemm_i8 import Case

pytestmark = pytest.mark.gpu


def give_up(M, N, K, add, d, units):
    c = Case(M, N, K, d, add=add, seed=M)
    want = c.run().d[:M, :N].clone()
    args = (c.a.data_ptr(), c.a.stride(0), c.sa.data_ptr(), c.w.data_ptr(), c.w.stride(0), c.sw.data_ptr(), c.d.data_ptr(), int(d == torch.bfloat16), c.ldd, M, N, K, int(add))
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    for unit in units:
        c.d.copy_(c.old)
        status.zero_()
        rc = lumi_b200.lib().lumi_debug_gemm_i8_wait_timeout(*args, 20_000_000, -2 - unit, status.data_ptr())
        got = c.d[:M, :N]
        lost = torch.isnan(got)
        assert rc == -7 and int(status) & 4 and bool(lost.any())
        assert torch.equal(got[~lost], want[~lost])
        assert torch.equal(c.d[M:], c.old[M:]) and torch.equal(c.d[:, N:], c.old[:, N:])
        c.d.copy_(c.old)
        assert torch.equal(c.run().d[:M, :N], want)


# one tile per CTA, with fewer and more k-blocks than stages; K shared by clusters
@pytest.mark.parametrize("M,N,K,add", [(64, 300, 256, False), (300, 520, 4096, True), (16, 1024, 2816, False), (40, 200, 8448, True)])
@pytest.mark.parametrize("d", [torch.float32, torch.bfloat16])
def test_tiles(M, N, K, add, d):
    give_up(M, N, K, add, d, [0, 1, 2])


# results by tensor-map copies (and old values of D the same way), and by single elements; several tiles per pair of CTAs: the first, a later and the last
@pytest.mark.parametrize("M,N,K,add", [(4096, 2560, 512, False), (4096, 7360, 256, True), (4100, 7361, 640, True), (9000, 5000, 130, False)])
@pytest.mark.parametrize("d", [torch.float32, torch.bfloat16])
def test_pairs(M, N, K, add, d):
    give_up(M, N, K, add, d, [0, 1, 75, 150])


@pytest.mark.parametrize("M,N,K,add", [(300, 520, 4096, True), (16, 1024, 2816, False), (4096, 7360, 256, True), (4100, 7361, 640, False)])
@pytest.mark.parametrize("limit", [1, 1000, 20_000])
def test_limits_that_are_too_short(M, N, K, add, limit):
    """What a call with a short limit clears up is waited for by the library's own limit: the call says whether a wait ran out, and the next one is right."""
    c = Case(M, N, K, add=add, seed=N)
    want = c.run().d[:M, :N].clone()
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    for _ in range(5):
        c.d.copy_(c.old)
        status.zero_()
        rc = lumi_b200.lib().lumi_debug_gemm_i8_wait_timeout(c.a.data_ptr(), c.a.stride(0), c.sa.data_ptr(), c.w.data_ptr(), c.w.stride(0), c.sw.data_ptr(), c.d.data_ptr(), 0, c.ldd,
                                                             M, N, K, int(add), limit, -1, status.data_ptr())
        lost = torch.isnan(c.d[:M, :N])
        assert rc == (-7 if bool(lost.any()) else 0) and torch.equal(c.d[:M, :N][~lost], want[~lost])
        c.d.copy_(c.old)
        assert torch.equal(c.run().d[:M, :N], want)
