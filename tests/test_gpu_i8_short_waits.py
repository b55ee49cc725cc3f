"""GPU: products in 8-bit integers whose waits on the device run out at any time, because their limit is far shorter than a copy takes.  Whichever of them do, the kernel ends
with its copies landed and its MMAs done, every result is the right one or NaN, nothing else is written, and the same product then runs as ever."""
import pytest
import torch

import lumi_b200
from tests.test_gpu_gemm_i8 import Case

pytestmark = pytest.mark.gpu


def run_short(M, N, K, add, d, limits):
    c = Case(M, N, K, d, add=add, seed=M)
    want = c.run().d[:M, :N].clone()
    args = (c.a.data_ptr(), c.a.stride(0), c.sa.data_ptr(), c.w.data_ptr(), c.w.stride(0), c.sw.data_ptr(), c.d.data_ptr(), int(d == torch.bfloat16), c.ldd, M, N, K, int(add))
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    for limit in limits:
        c.d.copy_(c.old)
        status.zero_()
        rc = lumi_b200.lib().lumi_debug_gemm_i8_wait_timeout(*args, limit, -1, status.data_ptr())
        got = c.d[:M, :N]
        lost = torch.isnan(got)
        assert rc == (-7 if int(status) & 4 else 0) and (rc != 0 or not bool(lost.any()))
        assert torch.equal(got[~lost], want[~lost])
        assert torch.equal(c.d[M:], c.old[M:]) and torch.equal(c.d[:, N:], c.old[:, N:])
    c.d.copy_(c.old)
    assert torch.equal(c.run().d[:M, :N], want)


@pytest.mark.parametrize("M,N,K,add", [(64, 300, 256, False), (300, 520, 4096, True), (16, 1024, 2816, False), (40, 200, 8448, True)])
@pytest.mark.parametrize("d", [torch.float32, torch.bfloat16])
def test_tiles(M, N, K, add, d):
    run_short(M, N, K, add, d, [1, 1, 500, 1000, 2000, 5000, 10000])
