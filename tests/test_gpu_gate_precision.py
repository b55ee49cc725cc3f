"""GPU: the gate in 8 bits (lumi_k_gate_quant), its numbers one by one: in rows of one number the scale is that number / 127.

Tolerances (u = 2^-24, a rounding to fp32).  fp32: expf is documented to be off by one ulp (2 u), an eighth of 1 + e^-v rounds once, the hardware's reciprocal is documented to be off by
one ulp (2 u), times gate and times up once each, / 127 once: 8 u, and where the sigmoid itself is no normal number half of 2^-149.  bf16: the exponent rounds once, which is u of
its size, |v| log2 e, times ln 2: |v| u; its constant is off by under u / 2 of it as well: 1.5 |v| u; ex2 is documented to be off by 2^-22.5 (2.9 u) and the sum, the reciprocal, the
products and / 127 as before: 1 + 2 + 2 + 1: 9 u."""
import pytest
import torch

import lumi_b200

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def scales(gate, up, act):
    n, dtype = gate.shape[0], gate.dtype
    gu = torch.zeros(n, 16, device="cuda", dtype=dtype)
    gu[:, 0], gu[:, 8] = gate, up
    q, s = torch.zeros(n, 16, device="cuda", dtype=torch.int8), torch.zeros(n, device="cuda")
    lumi_b200.api.check(lumi_b200.lib().lumi_k_gate_quant(gu.data_ptr(), int(dtype == torch.bfloat16), 16, 8, act, q.data_ptr(), 16, s.data_ptr(), n, 1, 0))
    torch.cuda.synchronize()
    return q[:, 0].double(), s.double()


@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("low,high", [(-4, 4), (4, 100), (-20, 0), (-60, -20), (-87, -60), (-88.5, -87.4)])
def test_gates_of_all_sizes(act, dtype, low, high):
    """Ups of 10^12, so that a closed gate's numbers are still above 2^-100."""
    n = 100_000
    g = torch.Generator(device="cuda").manual_seed(act)
    gate = (torch.rand(n, generator=g, device="cuda") * (high - low) + low).to(dtype)
    up = ((torch.rand(n, generator=g, device="cuda") + 1) * 1e12).to(dtype)
    q, s = scales(gate, up, act)
    z = gate.double()
    sigmoid = torch.sigmoid(z)
    t = sigmoid * up.double() * (z if act else 1)
    want = t.abs() / 127
    if dtype == torch.bfloat16 and high < -87.3:
        assert bool((q == 0).all())                       # closed
        return
    relative = 8 * U + 2.0 ** -150 / sigmoid if dtype == torch.float32 else (9 + 1.5 * z.abs()) * U
    assert float(((s - want).abs() / want - 1.01 * relative).max()) <= 0
    assert torch.equal(q, 127 * torch.sign(t))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gates_without_size(dtype):
    """Infinities, zeros and no number; far closed gates are zero, and so are the rows."""
    inf, nan = float("inf"), float("nan")
    gate = torch.tensor([inf, -inf, nan, 0.0, -0.0, -89.0, -1e30, 1e30, 100.0], device="cuda").to(dtype)
    up = torch.full((9,), 4.0, device="cuda").to(dtype)
    q, s = scales(gate, up, 0)
    assert q.tolist() == [127, 0, 0, 127, 127, 0, 0, 127, 127] and bool(torch.isnan(s[2]))
    assert float(s[0] * 127) == pytest.approx(4) and float(s[3] * 127) == pytest.approx(2) and float(s[1]) == pytest.approx(2.0 ** -100 / 127)
    q, s = scales(gate, up, 1)
    assert torch.isnan(s[:3]).all() and q.tolist()[3:] == [0, 0, 0, 0, 127, 127] and float(s[8] * 127) == pytest.approx(400)
