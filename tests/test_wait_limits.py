"""CPU: limits that the failure-path hooks of the bf16 products refuse, before a device is touched.  The kernels clear up within the same limit: below a millisecond, copies could still be under
way into shared memory that is given up.  Addresses are made up: none is looked at."""
import ctypes

import pytest

import lumi_b200
from lumi_b200.api import GemmProbe

P = 1 << 20


@pytest.mark.parametrize("limit", [1, 1000, 999_999])
def test_short_limits_are_refused(limit):
    L = lumi_b200.lib()
    assert L.lumi_debug_gemm_wait_timeout(P, P, P, 64, 64, 64, limit, -1, P) == -1
    assert b"wait limit" in L.lumi_last_error()
    p = GemmProbe(M=64, N=64, K=64, ldd=64, a_hi=P, w=P, d=P, skip_unit=-1, status_word=P, wait_limit_ns=limit)
    assert L.lumi_debug_gemm(ctypes.byref(p)) == -1
    assert b"wait limit" in L.lumi_last_error()
