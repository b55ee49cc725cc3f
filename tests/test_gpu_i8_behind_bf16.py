"""GPU: products in 8-bit integers directly behind bf16 products on the same stream (both allocate tensor memory, and the 8-bit one is launched while the other still runs), and the
other way round: the same bits as one by one, eager and captured."""
import pytest
import torch

import lumi_b200
from tests.test_gpu_gemm_i8 import Case

pytestmark = pytest.mark.gpu


class Bf16:
    def __init__(self, M, N, K, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.M, self.N, self.K = M, N, K
        self.a = torch.randn(M, K, generator=g, device="cuda").bfloat16()
        self.w = torch.randn(N, K, generator=g, device="cuda").bfloat16()
        self.d = torch.zeros(M, N, device="cuda")

    def call(self, stream=0):
        lumi_b200.api.check(lumi_b200.lib().lumi_k_gemm_bf16_tcgen05(self.a.data_ptr(), 0, self.w.data_ptr(), self.d.data_ptr(), self.M, self.N, self.K, self.N, 0, stream))


# single CTAs of several tile widths and pairs of CTAs, in front of tiles of 32 columns, of shares of K, and pairs
@pytest.mark.parametrize("M,N,K", [(300, 7360, 1024), (700, 2816, 512), (1024, 1536, 2048), (4096, 2048, 512)])
@pytest.mark.parametrize("m,n,k", [(20, 300, 256), (16, 1024, 2816), (300, 2000, 200), (4096, 2560, 256)])
def test_one_behind_the_other(M, N, K, m, n, k):
    b, c = Bf16(M, N, K, 1), Case(m, n, k, add=True, seed=2)
    b.call()
    torch.cuda.synchronize()
    want_b = b.d.clone()
    for _ in range(6):
        c.call()
    torch.cuda.synchronize()
    want_c = c.d.clone()

    def steps(stream):
        for i in range(6):
            b.call(stream)
            c.call(stream)

    for run in range(2):
        b.d.zero_(), c.d.copy_(c.old)
        torch.cuda.synchronize()
        if run == 0:
            s = torch.cuda.Stream()
            steps(s.cuda_stream)
        else:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=torch.cuda.Stream()):
                steps(torch.cuda.current_stream().cuda_stream)
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(b.d, want_b) and torch.equal(c.d, want_c)
