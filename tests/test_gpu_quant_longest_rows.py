"""GPU: rows as long as the calls on rows of 8-bit integers allow."""
import pytest
import torch

import lumi_b200

pytestmark = pytest.mark.gpu
LONGEST = 2 ** 30


def code(t):
    return 1 if t.dtype == torch.bfloat16 else 0


def places(width):
    """The first and last numbers of a row, and some around 2^29 and 2^30."""
    return [slice(0, 4096), slice(2 ** 29 - 2048, 2 ** 29 + 2048), slice(max(0, min(width, LONGEST) - 4096), width)]


@pytest.mark.parametrize("width", [LONGEST, LONGEST - 3])
def test_norm(width):
    """Tolerance of the scale: squares in chains of eight, added up in 64 bits, 10 levels of a tree; see the test of long rows: under 2^-19."""
    x = torch.ones(1, LONGEST, device="cuda", dtype=torch.bfloat16)
    x[0, 1::2] = -0.5
    x[0, width - 1] = 2.0
    w = torch.ones(LONGEST, device="cuda")
    q, s = torch.full((1, LONGEST), 99, device="cuda", dtype=torch.int8), torch.zeros(1, device="cuda")
    lumi_b200.api.check(lumi_b200.lib().lumi_k_norm_quant(x.data_ptr(), 1, LONGEST, 0, 0, 0, w.data_ptr(), q.data_ptr(), LONGEST, s.data_ptr(), 1, width, 1e-5, 0))
    torch.cuda.synchronize()
    squares = (width + 1) // 2 * 1.0 + width // 2 * 0.25 + 4.0 - (1.0 if width % 2 else 0.25)
    want = 2 / 127 / (squares / width + 1e-5) ** 0.5
    assert abs(float(s[0]) - want) <= 2.0 ** -19 * want
    assert bool((q[0, width:] == 99).all())
    for p in places(width):
        t = x[0, p].float()
        assert torch.equal(q[0, p].float(), torch.round(t * 63.5))          # 63.5 and 31.75: to 64 (even) and 32


@pytest.mark.parametrize("width", [LONGEST + 16, LONGEST + 13])
@pytest.mark.parametrize("shift", [0, 1])
def test_rows_back(width, shift):
    ld = LONGEST + 16
    q = torch.empty(1, ld, device="cuda", dtype=torch.int8)
    q.view(-1, 16)[:] = torch.arange(-8, 8, device="cuda", dtype=torch.int8)
    s = torch.tensor([0.75], device="cuda")
    whole = torch.full((ld + 8,), 7.0, device="cuda", dtype=torch.bfloat16)
    y = whole[shift:shift + ld].view(1, ld)
    lumi_b200.api.check(lumi_b200.lib().lumi_k_dequant_rows(q.data_ptr(), ld, s.data_ptr(), y.data_ptr(), 1, ld, 1, width, 0))
    torch.cuda.synchronize()
    for p in places(width):
        assert torch.equal(y[0, p], (q[0, p].float() * 0.75).bfloat16())
    assert bool((whole[:shift] == 7).all()) and bool((whole[shift + width:] == 7).all())
