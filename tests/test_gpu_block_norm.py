"""The norms around a block against 64 bits."""
import numpy as np
import pytest
import torch

import lumi_b200

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}          # of a rounding, relative
EPS = 1e-5


def rows_of(t, ld, dtype):
    buf = torch.full((t.shape[0], ld), float("nan"), device="cuda", dtype=dtype)
    buf[:, :t.shape[1]] = t.to("cuda").to(dtype)
    return buf


def call(x, o, post, gate, ldg, scale, pre, y, rows, width, eps=EPS, stream=None):
    code = lambda t: int(t is not None and t.dtype == BF16)
    ptr = lambda t: 0 if t is None else t.data_ptr()
    return lumi_b200.lib().lumi_k_block_norm(ptr(x), code(x), x.stride(0), ptr(o), code(o), o.stride(0), ptr(post), ptr(gate), ldg, scale, ptr(pre), ptr(y), code(y),
                                             0 if y is None else y.stride(0), rows, width, eps, torch.cuda.current_stream().cuda_stream if stream is None else stream)


def expected(x, o, post, gate, scale, pre, eps=EPS):
    """(new x before its rounding, its error's bound); y comes of the rounded x."""
    t = o.double()
    if post is not None:
        t = t / torch.sqrt((t * t).mean(1, keepdim=True) + eps) * post.double()
    if gate is not None:
        t = t * gate.double()
    # a dozen fp32 roundings of the added term (the sum of squares grows by at most log2(width) + 40 of them, half in its root) and one of the sum
    return x.double() + scale * t, (scale * t).abs() * 2.0 ** -19


def norm(x, pre, eps=EPS):
    t = x.double()
    return t / torch.sqrt((t * t).mean(1, keepdim=True) + eps) * pre.double()


@pytest.mark.parametrize("types", [(F32, F32, F32), (F32, BF16, BF16), (BF16, BF16, BF16), (BF16, F32, F32)])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (5, 8), (2, 100), (9, 256), (4, 300), (7, 512), (5, 1000), (6, 2048), (3, 4100), (2, 9999), (2, 16384), (2, 20003), (1, 32768)])
@pytest.mark.parametrize("form", ["rows", "one", "plain", "x alone"])
def test_rows(rows, width, types, form):
    xt, ot, yt = types
    g = torch.Generator().manual_seed(rows * 131 + width)
    rnd = lambda *s: torch.randn(*s, generator=g)
    ld = (width + 7) // 8 * 8 + 8
    x, o = rows_of(rnd(rows, width) * 3, ld, xt), rows_of(rnd(rows, width), ld, ot)
    post = None if form == "plain" else (1 + rnd(width) * 0.2).cuda()
    gate = None if form in ("plain", "x alone") else rows_of(rnd(1 if form == "one" else rows, width), ld, ot)
    pre = None if form == "x alone" else (1 + rnd(width) * 0.2).cuda()
    y = None if form == "x alone" else torch.full((rows, ld), -5.0, device="cuda", dtype=yt)
    want, slack = expected(x[:, :width], o[:, :width], post, None if gate is None else gate[:, :width], 0.7, pre)
    assert call(x, o, post, gate, 0 if form == "one" else ld, 0.7, pre, y, rows, width) == 0
    torch.cuda.synchronize()
    got = x[:, :width].double()
    assert ((got - want).abs() <= slack + (want.abs() + slack) * HALF[xt] + 2.0 ** -140).all()
    assert torch.isnan(x[:, width:]).all()
    if y is not None:
        exact = norm(x[:, :width], pre)
        assert ((y[:, :width].double() - exact).abs() <= exact.abs() * (2.0 ** -19 + HALF[yt]) + 2.0 ** -140).all()
        assert (y[:, width:] == -5.0).all()


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e18, 3e37])
def test_rows_of_any_size(size):
    """Squares leave fp32's range on either side; eps is tiny, so the norm is what it would be at size one."""
    g = torch.Generator().manual_seed(1)
    width = 777
    o = rows_of(torch.randn(3, width, generator=g) * size, 784, F32)
    x = rows_of(torch.zeros(3, width), 784, F32)
    one = torch.ones(width, device="cuda")
    y = torch.zeros(3, 784, device="cuda")
    assert call(x, o, one, None, 0, 1.0, one, y, 3, width, eps=1e-37) == 0
    t = o[:, :width].double()
    want = t / torch.sqrt((t * t).mean(1, keepdim=True) + 1e-37)
    assert ((x[:, :width].double() - want).abs() <= want.abs() * 2.0 ** -18).all()


def test_rows_that_are_no_numbers_stay_alone():
    x, o = torch.randn(4, 64, device="cuda"), torch.randn(4, 64, device="cuda")
    before = x.clone()
    alone = before[3:].clone()
    o[1, 5], o[2, 7] = float("nan"), float("inf")
    one, y = torch.ones(64, device="cuda"), torch.zeros(4, 64, device="cuda")
    assert call(x, o, one, None, 0, 1.0, one, y, 4, 64) == 0
    y1 = torch.zeros(1, 64, device="cuda")
    assert call(alone, o[3:], one, None, 0, 1.0, one, y1, 1, 64) == 0
    assert torch.isnan(y[1]).all() and torch.isnan(x[1]).all()
    assert torch.isnan(x[2, 7]) and torch.equal(x[2, :7], before[2, :7])            # the others over an infinite norm: nothing is added
    assert torch.equal(y[3:], y1) and torch.equal(x[3:], alone)
    zero = torch.zeros(2, 64, device="cuda")
    assert call(zero, torch.zeros(2, 64, device="cuda"), one, None, 0, 1.0, one, y, 2, 64) == 0
    assert (zero == 0).all() and (y[:2] == 0).all()


def test_captured_and_on_another_stream():
    x, o = torch.randn(40, 1024, device="cuda"), torch.randn(40, 1024, device="cuda")
    one, y = torch.ones(1024, device="cuda"), torch.zeros(40, 1024, device="cuda", dtype=BF16)
    want = x.clone()
    for _ in range(3):
        want = (want.double() + o.double() / torch.sqrt((o.double() ** 2).mean(1, keepdim=True) + EPS)).float()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            assert call(x, o, one, None, 0, 1.0, one, y, 40, 1024, stream=side.cuda_stream) == 0
        for _ in range(3):
            graph.replay()
    side.synchronize()
    assert (x - want).abs().max() <= 8 * 2.0 ** -20
