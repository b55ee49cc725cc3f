"""GPU: rows of millions of numbers in 8 bits, against 64 bits.

Tolerance of a norm's scale (u = 2^-24, a rounding to fp32).  Up to 65536 numbers: a thread's squares are a chain of 64 (64 u of a sum of positive terms), a row's last numbers add once,
and 10 levels of a tree are left: 75 u, halved by the root; the quotient, the sum with eps, root, reciprocal, m / 127 and the last product once each, the product x w of the largest
once: under 45 u, below 2^-18.  Beyond: chains of eight, added up in 64 bits and rounded once, the rest the same: 20 u, halved, and 7: under 17 u, below 2^-19.  In a scaled second pass
the product with a power of two is exact."""
import pytest
import torch

import lumi_b200

pytestmark = pytest.mark.gpu
EPS = 1e-5


def scale_of(x, o, w, width, eps=EPS):
    q = torch.zeros(x.shape[0], x.stride(0), device="cuda", dtype=torch.int8)
    s = torch.zeros(x.shape[0], device="cuda")
    lumi_b200.api.check(lumi_b200.lib().lumi_k_norm_quant(x.data_ptr(), int(x.dtype == torch.bfloat16), x.stride(0), 0 if o is None else o.data_ptr(), 0 if o is None else int(o.dtype == torch.bfloat16),
                                                          0 if o is None else o.stride(0), w.data_ptr(), q.data_ptr(), x.stride(0), s.data_ptr(), x.shape[0], width, eps, 0))
    torch.cuda.synchronize()
    return q, s


@pytest.mark.parametrize("width", [20001, 65536, 65537, 1 << 20, (1 << 22) + 5, 1 << 26])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", [1.1, 1.9, None])
def test_sums_of_squares(width, dtype, value):
    """Equal numbers round the same way at every addition; and normal ones."""
    ld = (width + 15) // 16 * 16
    if value is None:
        x = torch.randn(1, ld, device="cuda", generator=torch.Generator(device="cuda").manual_seed(width)).to(dtype)
    else:
        x = torch.full((1, ld), value, device="cuda", dtype=dtype)
    w = torch.ones(ld, device="cuda")
    q, s = scale_of(x, None, w, width)
    t = x[:, :width].double()
    m = t.abs().amax()
    want = m / 127 / torch.sqrt((t * t).mean() + EPS)
    assert abs(float(s[0]) - float(want)) <= 2.0 ** (-18 if width <= 65536 else -19) * float(want)
    assert float((q[0, :width].double() - t[0] * 127 / m).abs().max()) <= 0.5 + 127 * 2.0 ** -21


@pytest.mark.parametrize("size,eps", [(1e30, 1e-5), (1e-25, 1e-37)])
def test_squares_out_of_range(size, eps):
    """Sums that overflow, or vanish beside a small eps, are taken again of scaled numbers, as closely."""
    width = 1 << 22
    x = torch.full((2, width), 1.3 * size, device="cuda")
    q, s = scale_of(x, None, torch.ones(width, device="cuda"), width, eps)
    t = x[0, 0].double()
    want = t / 127 / torch.sqrt(t * t + float(torch.tensor(eps)))
    assert float((s.double() - want).abs().max()) <= 2.0 ** -19 * float(want) and bool((q == 127).all())


def test_with_a_residual():
    width = (1 << 22) + 16
    x, o = torch.full((1, width), 0.7, device="cuda"), torch.full((1, width), 0.4, device="cuda", dtype=torch.bfloat16)
    t = (x[0, 0] + o[0, 0].float()).double()
    q, s = scale_of(x, o, torch.ones(width, device="cuda"), width)
    want = t / 127 / torch.sqrt(t * t + EPS)
    assert bool((x.double() == t).all()) and bool((q[:, :width] == 127).all()) and abs(float(s[0]) - float(want)) <= 2.0 ** -19 * float(want)
