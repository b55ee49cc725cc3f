"""GPU: calls on rows of 8-bit integers by several host threads at once, of which every single one has to have run."""
import threading

import pytest
import torch

import lumi_b200
from tests.test_gpu_gemm_i8 import Case

pytestmark = pytest.mark.gpu
CALLS = 20


def test_every_threads_every_call():
    """D holds something else before, and every call adds to it, so that one that did nothing would be seen; each thread is compared with as many calls one by one."""
    cases = [Case(M, 1024, 1024, [torch.float32, torch.bfloat16][M % 2], add=True, seed=M) for M in (1, 7, 30, 500, 4096)]
    want = []
    for c in cases:
        for _ in range(CALLS):
            c.call()
        torch.cuda.synchronize()
        want.append(c.d.clone())
        c.d.copy_(c.old)
        assert not torch.equal(c.old, want[-1])
    torch.cuda.synchronize()
    same = [False] * len(cases)
    start = threading.Barrier(len(cases))

    def work(i):
        stream = torch.cuda.Stream()
        start.wait()
        for _ in range(CALLS):
            cases[i].call(stream.cuda_stream)
        stream.synchronize()
        same[i] = torch.equal(cases[i].d, want[i])

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(same)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_several_threads(dtype):
    """Norms that add a residual, and gates, each thread's on a stream of its own; the stream's rows grow with every call."""
    g = torch.Generator(device="cuda").manual_seed(1)
    L, ok, bf = lumi_b200.lib(), lumi_b200.api.check, int(dtype == torch.bfloat16)
    sets = []
    for width in (96, 1000, 2816, 20000):
        x0, o = (torch.randn(300, (width + 15) // 16 * 16, generator=g, device="cuda").to(dtype) for _ in range(2))
        sets.append((width, x0, o, x0.clone(), torch.zeros(300, x0.stride(0), device="cuda", dtype=torch.int8), torch.zeros(300, device="cuda")))

    def calls(width, x0, o, x, q, s, stream):
        for _ in range(CALLS):
            ok(L.lumi_k_norm_quant(x.data_ptr(), bf, x.stride(0), o.data_ptr(), bf, o.stride(0), 0, q.data_ptr(), q.stride(0), s.data_ptr(), 300, width, 0.0, stream))

    want = []
    for t in sets:
        calls(*t, 0)
        torch.cuda.synchronize()
        want.append([u.clone() for u in t[3:]])
        t[3].copy_(t[1]), t[4].fill_(99), t[5].fill_(-1)
        assert not torch.equal(t[3], want[-1][0])
    torch.cuda.synchronize()
    same = [False] * len(sets)

    def work(i):
        stream = torch.cuda.Stream()
        calls(*sets[i], stream.cuda_stream)
        stream.synchronize()
        w = sets[i][0]
        x, q, s = sets[i][3:]
        same[i] = torch.equal(x, want[i][0]) and torch.equal(q[:, :w], want[i][1][:, :w]) and torch.equal(s, want[i][2])

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sets))]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(same)


@pytest.mark.parametrize("width", [96, 704, 1000, 2048, 4096, 8200, 16384, 20000])
@pytest.mark.parametrize("x_dtype,o_dtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
def test_a_row_alone_and_among_others_with_a_residual(width, x_dtype, o_dtype):
    """Where blocks take row after row (a bf16 stream with its residual) a row's bits are still its own: more rows than run at once, their order turned round, and single ones."""
    g = torch.Generator(device="cuda").manual_seed(width)
    rows = 3000 if width <= 8200 else 1200
    ld = (width + 15) // 16 * 16
    x0 = torch.randn(rows, ld, generator=g, device="cuda").to(x_dtype)
    o = torch.randn(rows, ld, generator=g, device="cuda").to(o_dtype)
    w = torch.randn(ld, generator=g, device="cuda")

    def norm(x, o):
        x, n = x.clone(), x.shape[0]
        q, s = torch.zeros(n, ld, device="cuda", dtype=torch.int8), torch.zeros(n, device="cuda")
        lumi_b200.api.check(lumi_b200.lib().lumi_k_norm_quant(x.data_ptr(), int(x_dtype == torch.bfloat16), ld, o.data_ptr(), int(o_dtype == torch.bfloat16), ld, w.data_ptr(), q.data_ptr(), ld,
                                                              s.data_ptr(), n, width, 1e-5, 0))
        torch.cuda.synchronize()
        return x[:, :width], q[:, :width], s

    all_of = norm(x0, o)
    back = norm(x0.flip(0), o.flip(0))
    assert all(torch.equal(a, b.flip(0)) for a, b in zip(all_of, back))
    for r in (0, 1, rows // 2, rows - 1):
        assert all(torch.equal(a[r:r + 1], b) for a, b in zip(all_of, norm(x0[r:r + 1], o[r:r + 1])))
