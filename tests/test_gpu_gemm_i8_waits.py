"""GPU: bounded device waits of the products in 8-bit integers.  A tile's operands never arrive; its waits run out, the kernel returns by itself, the results that this
cost are NaN and no others, and the same product then runs as ever.  Nothing is faulted: a wait is merely never answered."""
import pytest
import torch

import lumi_b200
from tests.test_gpu_gemm_i8 import Case

pytestmark = pytest.mark.gpu


# one tile per CTA; K shared by clusters; pairs of CTAs, results by tensor-map copies and by single elements
@pytest.mark.parametrize("M,N,K,add", [(64, 300, 256, False), (300, 520, 512, True), (16, 1024, 2816, False), (40, 200, 8448, True),
                                       (4096, 2560, 512, False), (4096, 2560, 512, True), (4100, 2561, 640, True)])
@pytest.mark.parametrize("skip", [0, 1, 3])
def test_lost_wait(M, N, K, add, skip):
    for d in (torch.float32, torch.bfloat16):
        c = Case(M, N, K, d, add=add, seed=skip)
        want = c.run().d[:M, :N].clone()
        c.d.copy_(c.old)
        status = torch.zeros(1, device="cuda", dtype=torch.int32)
        args = (c.a.data_ptr(), c.a.stride(0), c.sa.data_ptr(), c.w.data_ptr(), c.w.stride(0), c.sw.data_ptr(), c.d.data_ptr(), int(d == torch.bfloat16), c.ldd, M, N, K, int(add))
        rc = lumi_b200.lib().lumi_debug_gemm_i8_wait_timeout(*args, 2_000_000, skip, status.data_ptr())
        assert rc == -7 and int(status) & 4
        got = c.d[:M, :N]
        lost = torch.isnan(got)
        assert 0 < int(lost.sum()) and torch.equal(got[~lost], want[~lost])
        assert torch.equal(c.d[M:], c.old[M:]) and torch.equal(c.d[:, N:], c.old[:, N:])
        status.zero_()
        c.d.copy_(c.old)
        assert lumi_b200.lib().lumi_debug_gemm_i8_wait_timeout(*args, 500_000_000, -1, status.data_ptr()) == 0
        assert torch.equal(c.d[:M, :N], want)
        c.d.copy_(c.old)
        assert torch.equal(c.run().d[:M, :N], want)
