"""GPU: products in 8-bit integers (lumi_k_gemm_i8) against the definition in 64 bits (sums of products of 8-bit integers are whole numbers below 2^53, which
64-bit floating products hold exactly).

Tolerance: the sum is exact; u = 2^-24.  Its way to fp32 and the products with the two scales round once each (3 u of the product), adding the bias and
the old value once each (u of the sum), a bf16 result once more (2^-8 of it): see `allowed`."""
import itertools

import pytest
import torch

import lumi_b200

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def up(n, k=16):
    return (n + k - 1) // k * k


def codes(g, rows, width, pad=0, low=-128, high=128):
    """8-bit rows; what lies between them would count."""
    buf = torch.full((rows, up(width) + pad), 77, device="cuda", dtype=torch.int8)
    buf[:, :width] = torch.randint(low, high, (rows, width), generator=g, device="cuda", dtype=torch.int16).to(torch.int8)
    return buf


class Case:
    def __init__(self, M, N, K, d=torch.float32, bias=False, add=False, pad=0, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.M, self.N, self.K, self.add = M, N, K, add
        self.a, self.w = codes(g, M, K, pad), codes(g, N, K, 2 * pad)
        self.sa = torch.rand(M, generator=g, device="cuda") + 0.5
        self.sw = (torch.rand(N, generator=g, device="cuda") + 0.5) * 1e-3
        self.b = torch.randn(N, generator=g, device="cuda") * 30 if bias else None
        self.ldd = N + (pad and 3)
        self.d = torch.full((M + 1, self.ldd), -5.0, device="cuda", dtype=d)
        self.d[:M, :N] = torch.randn(M, N, generator=g, device="cuda") * 30
        self.old = self.d.clone()

    def args(self, stream=0, status=0):
        return (self.a.data_ptr(), self.a.stride(0), self.sa.data_ptr(), self.w.data_ptr(), self.w.stride(0), self.sw.data_ptr(),
                0 if self.b is None else self.b.data_ptr(), self.d.data_ptr(), int(self.d.dtype == torch.bfloat16), self.ldd, self.M, self.N, self.K,
                int(self.add), status, stream)

    def call(self, stream=0, status=0):
        lumi_b200.api.check(lumi_b200.lib().lumi_k_gemm_i8(*self.args(stream, status)))

    def run(self):
        self.call()
        torch.cuda.synchronize()
        return self

    def want(self):
        p = (self.a[:, :self.K].double() @ self.w[:, :self.K].double().t()) * self.sa.double()[:, None] * self.sw.double()
        q = p + self.b.double() if self.b is not None else p
        r = q + self.old[:self.M, :self.N].double() if self.add else q
        allowed = 3.01 * U * p.abs() + 1.01 * U * (q.abs() + r.abs())
        if self.d.dtype == torch.bfloat16:
            allowed += 1.01 * 2.0 ** -8 * r.abs()
        return r, allowed

    def check(self):
        r, allowed = self.want()
        far = (self.d[:self.M, :self.N].double() - r).abs() - allowed
        assert float(far.max()) <= 0, (self.M, self.N, self.K, float(far.max()))
        assert torch.equal(self.d[self.M:], self.old[self.M:]) and torch.equal(self.d[:, self.N:], self.old[:, self.N:])


FORMS = list(itertools.product([torch.float32, torch.bfloat16], [False, True], [False, True]))


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 48, 64, 65, 100, 127, 128, 129, 200, 255, 256, 257, 384, 500, 777, 1024, 2049])
def test_rows(M):
    for i, (N, K) in enumerate([(1, 1), (5, 17), (31, 16), (128, 128), (130, 1111), (259, 1024), (1024, 96), (2053, 640), (7360, 129)]):
        d, bias, add = FORMS[(i + M) % 8]
        Case(M, N, K, d, bias, add, pad=16 * (i % 2), seed=i).run().check()


@pytest.mark.parametrize("K", [1, 2, 15, 16, 31, 33, 64, 100, 127, 128, 129, 255, 257, 1000, 1024, 2816, 4096, 8448, 16385, 65537])
def test_lengths(K):
    for i, (M, N) in enumerate([(1, 100), (6, 259), (16, 1024), (40, 130), (130, 257), (300, 520)]):
        d, bias, add = FORMS[(i + K) % 8]
        Case(M, N, K, d, bias, add, pad=32 * (i % 2), seed=i).run().check()


@pytest.mark.parametrize("d,bias,add", FORMS)
def test_large(d, bias, add):
    """Many tiles of the largest kind, whole and with remainders on every side."""
    Case(4096, 2048, 1024, d, bias, add).run().check()
    Case(4111, 4099, 1555, d, bias, add, pad=16).run().check()
    Case(9000, 300, 513, d, bias, add).run().check()
    Case(300, 9000, 513, d, bias, add).run().check()


@pytest.mark.parametrize("M,N,K", [(1, 77, 200), (5, 77, 200), (30, 300, 1000), (30, 300, 3000), (5000, 520, 200)])
@pytest.mark.parametrize("d", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1])
def test_operands_that_begin_and_end_anywhere(M, N, K, d, shift):
    """Bases 16 bytes behind a larger boundary, operands that end with their last number, results that begin at any element."""
    g = torch.Generator(device="cuda").manual_seed(M + shift)
    ld = up(K)

    def rows(n):
        buf = torch.full((16 + (n - 1) * ld + K,), 99, device="cuda", dtype=torch.int8)
        t = buf[16:].as_strided((n, K), (ld, 1))
        t.copy_(torch.randint(-128, 128, (n, K), generator=g, device="cuda", dtype=torch.int16).to(torch.int8))
        return t

    a, w = rows(M), rows(N)
    sa, sw, b = (torch.rand(n + 1, generator=g, device="cuda")[1:] for n in (M, N, N))
    old = torch.randn(M * N + shift + 1, generator=g, device="cuda").to(d)
    for add in (0, 1):
        whole = old.clone()
        out = whole[shift:shift + M * N].view(M, N)
        lumi_b200.api.check(lumi_b200.lib().lumi_k_gemm_i8(a.data_ptr(), ld, sa.data_ptr(), w.data_ptr(), ld, sw.data_ptr(), b.data_ptr(), out.data_ptr(),
                                                           int(d == torch.bfloat16), N, M, N, K, add, 0, 0))
        torch.cuda.synchronize()
        p = (a.double() @ w.double().t()) * sa.double()[:, None] * sw.double()
        q = p + b.double()
        r = q + (old[shift:shift + M * N].view(M, N).double() if add else 0)
        allowed = 3.01 * U * p.abs() + 1.01 * U * (q.abs() + r.abs()) + (1.01 * 2.0 ** -8 * r.abs() if d == torch.bfloat16 else 0)
        assert float(((out.double() - r).abs() - allowed).max()) <= 0
        assert torch.equal(whole[:shift], old[:shift]) and torch.equal(whole[shift + M * N:], old[shift + M * N:])


@pytest.mark.parametrize("M,N", [(1, 7), (3, 40), (20, 130), (300, 300)])
def test_largest_sums(M, N):
    """131071 products of -128 and -128: 2^31 - 2^14."""
    K = 131071
    c = Case(M, N, K)
    c.a[:, :K], c.w[:, :K] = -128, -128
    c.sa[:], c.sw[:] = 1, 1
    c.run()
    assert bool((c.d[:M, :N].double() == 2.0 ** 31 - 2.0 ** 14).all())
    c.w[:, :K] = 127
    c.run()
    assert bool((c.d[:M, :N].double() == float(torch.tensor(-128.0 * 127 * K))).all())


@pytest.mark.parametrize("M,N,K", [(1, 300, 256), (24, 300, 2048), (700, 2000, 512), (5000, 2000, 256)])
def test_rows_without_numbers(M, N, K):
    """A scale that is NaN, infinite or zero is that row's or column's alone."""
    c = Case(M, N, K)
    c.sa[M - 1] = float("nan")
    c.sw[5], c.sw[7] = float("nan"), 0
    c.run()
    got = c.d[:M, :N]
    assert bool(torch.isnan(got[M - 1]).all()) and bool(torch.isnan(got[:, 5]).all())
    if M > 1:
        assert bool((got[:M - 1, 7] == 0).all())
        keep = [n for n in range(N) if n != 5]
        r, allowed = c.want()
        assert float(((got.double() - r).abs() - allowed)[:M - 1][:, keep].max()) <= 0


def test_same_bits_again():
    for M, N, K in ((1, 7360, 1024), (16, 1024, 2816), (203, 2053, 1111), (1000, 1024, 2048), (4096, 2048, 512)):
        c = Case(M, N, K)
        first = c.run().d.clone()
        c.d.copy_(c.old)
        assert torch.equal(c.run().d, first)


def test_rows_in_a_wide_buffer():
    """Rows of A, W and D beyond 2^31 elements from the first."""
    g = torch.Generator(device="cuda").manual_seed(7)
    rows, ld = 2200, 1 << 20
    a = torch.empty(rows * ld, device="cuda", dtype=torch.int8).view(rows, ld)       # 2.3 GB
    a[:, :128] = codes(g, rows, 128)
    d = torch.empty(rows * ld, device="cuda", dtype=torch.bfloat16).view(rows, ld)   # 4.6 GB
    w = codes(g, rows, 128)
    one = torch.ones(rows, device="cuda")
    call = lumi_b200.lib().lumi_k_gemm_i8
    for M, N, args in ((rows, 64, (a.data_ptr(), ld, w.data_ptr(), 128)), (64, rows, (w.data_ptr(), 128, a.data_ptr(), ld)), (3, rows, (w.data_ptr(), 128, a.data_ptr(), ld))):
        lumi_b200.api.check(call(args[0], args[1], one.data_ptr(), args[2], args[3], one.data_ptr(), 0, d.data_ptr(), 1, ld, M, N, 128, 0, 0, 0))
        torch.cuda.synchronize()
        x, y = (a, w) if args[1] == ld else (w, a)
        want = x[:M, :128].double() @ y[:N, :128].double().t()
        assert float(((d[:M, :N].double() - want).abs() - 2.0 ** -8 * want.abs()).max()) <= 0


def test_streams_and_graphs():
    """Calls on two streams at once, and two captured graphs replayed beside one another, give what calls one by one give."""
    cases = [Case(8, 1024, 2816, seed=1), Case(64, 1024, 2816, seed=2), Case(600, 1024, 2048, seed=3), Case(4096, 2048, 1024, torch.bfloat16, seed=4)]
    want = [c.run().d.clone() for c in cases]
    for c in cases:
        c.d.copy_(c.old)
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        for c, s in zip(cases, streams):
            c.call(s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(c.d, w) for c, w in zip(cases, want))
    graphs = []
    for c, s in zip(cases, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            c.call(torch.cuda.current_stream().cuda_stream)
            c.call(torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for c in cases:
        c.d.copy_(c.old)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(c.d, w) for c, w in zip(cases, want))


class Mlp:
    """A feed-forward in 8 bits behind a residual: x += o; norm; gate and up; gate; down into x."""

    def __init__(self, rows, width, ff, act, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
        self.rows, self.width, self.ff, self.act = rows, width, ff, act
        self.x, self.o, self.g = rand(rows, width), rand(rows, width).bfloat16(), 1 + 0.1 * rand(width)
        self.x0 = self.x.clone()
        self.w1, self.w2 = rand(2 * ff, width).bfloat16() / width ** 0.5, rand(width, ff).bfloat16() / ff ** 0.5
        byte = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int8)
        self.q1, self.s1, self.q2, self.s2 = byte(2 * ff, width), torch.zeros(2 * ff, device="cuda"), byte(width, ff), torch.zeros(width, device="cuda")
        self.a, self.sa, self.h, self.sh = byte(rows, width), torch.zeros(rows, device="cuda"), byte(rows, ff), torch.zeros(rows, device="cuda")
        self.gu = torch.zeros(rows, 2 * ff, device="cuda", dtype=torch.bfloat16)
        L, ok = lumi_b200.lib(), lumi_b200.api.check
        for w, q, s in ((self.w1, self.q1, self.s1), (self.w2, self.q2, self.s2)):
            ok(L.lumi_k_norm_quant(w.data_ptr(), 1, w.shape[1], 0, 0, 0, 0, q.data_ptr(), w.shape[1], s.data_ptr(), w.shape[0], w.shape[1], 0.0, 0))

    def run(self, stream):
        L, ok, p = lumi_b200.lib(), lumi_b200.api.check, (lambda t: t.data_ptr())
        r, n, f = self.rows, self.width, self.ff
        ok(L.lumi_k_norm_quant(p(self.x), 0, n, p(self.o), 1, n, p(self.g), p(self.a), n, p(self.sa), r, n, 1e-5, stream))
        ok(L.lumi_k_gemm_i8(p(self.a), n, p(self.sa), p(self.q1), n, p(self.s1), 0, p(self.gu), 1, 2 * f, r, 2 * f, n, 0, 0, stream))
        ok(L.lumi_k_gate_quant(p(self.gu), 1, 2 * f, f, self.act, p(self.h), f, p(self.sh), r, f, stream))
        ok(L.lumi_k_gemm_i8(p(self.h), f, p(self.sh), p(self.q2), f, p(self.s2), 0, p(self.x), 0, n, r, n, f, 1, 0, stream))


@pytest.mark.parametrize("rows,act", [(1, 0), (5, 1), (48, 1), (700, 0), (4100, 1)])
def test_feed_forward(rows, act):
    """The four calls one behind another, eager and captured.  Against the same feed-forward in 64 bits without 8-bit steps: rounding to 8 bits moves a
    number by at most half its row's step.  A row of normal numbers has a largest of at most 6 (rows of at most 2816 numbers; the values here are
    fixed by their seeds), so a step is at most 6 / 127, and its error, uniform, 6 / 127 / sqrt(12) = 1.4 % of the row's root mean square, in each of the
    four quantised operands and twice more through the gate's product (its rows have a largest of at most 20 times their root mean square: 4.6 %), the
    bf16 rows of gate and up 0.2 %: root of the sum of squares 1.4 (x 4), 4.6, 0.2: under 6 %."""
    width, ff = 1024, 2816
    m = Mlp(rows, width, ff, act)
    m.run(0)
    torch.cuda.synchronize()
    eager = m.x.clone()
    x = m.x0.double() + m.o.double()
    y = x / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-5) * m.g.double()
    gu = y @ m.w1.double().t()
    h = torch.sigmoid(gu[:, :ff]) * gu[:, ff:] * (gu[:, :ff] if act else 1)
    out = h @ m.w2.double().t()
    got = eager.double() - x
    assert float((got - out).norm() / out.norm()) < 0.06
    # and exactly, from what the kernels left between them
    p = (m.h.double() @ m.q2.double().t()) * m.sh.double()[:, None] * m.s2.double()
    old = (m.x0 + m.o.float()).double()
    assert float(((eager.double() - (old + p)).abs() - (3.01 * U * p.abs() + 1.01 * U * ((old + p).abs()))).max()) <= 0
    p = (m.a.double() @ m.q1.double().t()) * m.sa.double()[:, None] * m.s1.double()
    assert float(((m.gu.double() - p).abs() - 1.01 * 2.0 ** -8 * p.abs()).max()) <= 0
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        m.run(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        m.x.copy_(m.x0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(m.x, eager)
