"""GPU: the calls on rows of 8-bit integers in a process whose first call is inside a stream capture, on a device that has nothing of them loaded; a chain replayed on changed
inputs; and calls of several host threads at once."""
import subprocess
import sys
import threading

import pytest
import torch

import lumi_b200
from tests.test_gpu_gemm_i8 import Case, Mlp

pytestmark = pytest.mark.gpu

FIRST = """
import torch, lumi_b200
from tests.test_gpu_gemm_i8 import Case, Mlp
lumi_b200.lib()
cases = [Case(1, 300, 256), Case(8, 300, 256), Case(20, 1024, 2816), Case(64, 300, 256), Case(4096, 2560, 256, add=True)]
q = torch.zeros(5, 1024, device="cuda", dtype=torch.int8)
s, y = torch.zeros(5, device="cuda"), torch.zeros(5, 1024, device="cuda")
x = torch.randn(5, 1024, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    stream = torch.cuda.current_stream().cuda_stream
    for c in cases:
        c.call(stream)
    lumi_b200.api.check(lumi_b200.lib().lumi_k_norm_quant(x.data_ptr(), 0, 1024, 0, 0, 0, 0, q.data_ptr(), 1024, s.data_ptr(), 5, 1024, 0.0, stream))
    lumi_b200.api.check(lumi_b200.lib().lumi_k_dequant_rows(q.data_ptr(), 1024, s.data_ptr(), y.data_ptr(), 0, 1024, 5, 1024, stream))
g.replay()
torch.cuda.synchronize()
for c in cases:
    c.check()
assert float((y - x).abs().max()) <= float(s.max()) * 0.501
print("captured")
"""


def test_first_call_inside_a_capture():
    out = subprocess.run([sys.executable, "-c", FIRST], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]


def test_replayed_on_other_inputs():
    """A captured feed-forward reads what its buffers hold at each replay."""
    m = Mlp(9, 512, 704, 1)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        m.run(torch.cuda.current_stream().cuda_stream)
    for seed in (1, 2):
        x = torch.randn(9, 512, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
        m.x.copy_(x)
        g.replay()
        torch.cuda.synchronize()
        got = m.x.clone()
        m.x.copy_(x)
        m.run(0)
        torch.cuda.synchronize()
        assert torch.equal(got, m.x)


def test_host_threads():
    """Calls of several threads, each on a stream of its own, and a refused one among them whose message is its thread's alone."""
    cases = [Case(M, 1024, 1024, seed=M) for M in (1, 7, 30, 500, 4096)]
    want = [c.run().d.clone() for c in cases]
    said = []

    def work(c, w):
        stream = torch.cuda.Stream()
        for _ in range(20):
            c.call(stream.cuda_stream)
        bad = lumi_b200.lib().lumi_k_gemm_i8(0, *c.args(stream.cuda_stream)[1:])
        said.append((bad, b"lumi_k_gemm_i8" in lumi_b200.lib().lumi_last_error()))
        stream.synchronize()
        said.append(torch.equal(c.d, w))

    threads = [threading.Thread(target=work, args=a) for a in zip(cases, want)]
    torch.cuda.synchronize()
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert len(said) == 10 and all(x is True or x == (-1, True) for x in said)
