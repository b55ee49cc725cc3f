"""Attention over the cache in 4 bits when a wait of its kernels gives up: a page that never arrives."""
import pytest
import torch

import lumi_b200
from tests.test_gpu_kv4_attention import BF16, F32, Batch

pytestmark = pytest.mark.gpu


def hook(b, skip, limit_ns):
    return lumi_b200.lib().lumi_debug_kv4_attention_wait_timeout(
        b.q.data_ptr(), b.q.stride(0), int(b.dtype == BF16), b.kv.data_ptr(), b.n_pages, b.d_table.data_ptr(), b.width, b.d_start.data_ptr(), b.d_tokens.data_ptr(), b.y.data_ptr(),
        b.y.stride(0), b.heads, b.kv_heads, b.dk, b.dv, 0, b.dk ** -0.5, 0, len(b.held), b.rows, max(b.new), b.work.data_ptr(), b.work.numel(), b.status.data_ptr(), limit_ns, skip)


# (new rows of each sequence, the page that does not arrive, the sequence it is of: a step's sequences have 10, 15 and 11 pages, prompts' begin with three places, the first one's 14 in all)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,skip,of", [((1, 1, 1), 0, 0), ((1, 1, 1), 20, 1), ((2, 1, 1), 10 + 15 + 5, 2), ((60, 80, 40), 3, 0), ((60, 80, 40), 14 + 3 + 5, 1)])
def test_a_page_that_does_not_arrive(new, skip, of, d, dtype):
    """The call comes back with the status, rows that the page costs are NaN, the others are NaN or right; the next call with the same work area is right."""
    held = [600, 900, 700]
    b = Batch(held, new, 2, 1, d, d, dtype)
    torch.cuda.synchronize()
    assert hook(b, skip, 3_000_000) == -7 and int(b.status) == 4
    first = b.y.clone()
    assert torch.isnan(first[b.starts[of]:b.starts[of + 1], :2 * d]).any()
    assert (first[b.rows:] == -5.0).all()
    b.status.zero_()
    b.y.fill_(-5.0)
    torch.cuda.synchronize()
    b.check()
    lost = torch.isnan(first)
    close = (first.float() - b.y.float()).abs() <= 2.0 ** (-6 if dtype == BF16 else -14)
    assert (lost | close)[:b.rows].all()
    b.y.fill_(-5.0)
    torch.cuda.synchronize()
    assert hook(b, -1, 2_000_000_000) == 0
    b.check(run=False)
