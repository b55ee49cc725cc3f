"""CPU: what the calls on rows of 8-bit integers refuse, and that they refuse it before a device is touched.  Addresses are made up: none is looked at."""
import pytest

import lumi_b200

INVALID, UNSUPPORTED, CUDA = -1, -10, -6
P = 1 << 20      # an address on a 16-byte boundary


def norm(**k):
    a = dict(x=P, x_dtype=0, ldx=64, o=P, o_dtype=0, ldo=64, w=P, q=P, ldq=64, scale=P, rows=0, width=64, eps=1e-5, stream=0)
    assert set(k) <= set(a)
    return lumi_b200.lib().lumi_k_norm_quant(*{**a, **k}.values())


def gate(**k):
    a = dict(gu=P, dtype=0, ld=128, up=64, act=0, q=P, ldq=64, scale=P, rows=0, width=64, stream=0)
    assert set(k) <= set(a)
    return lumi_b200.lib().lumi_k_gate_quant(*{**a, **k}.values())


def dequant(**k):
    a = dict(q=P, ldq=64, scale=P, y=P, y_dtype=0, ldy=64, rows=0, width=64, stream=0)
    assert set(k) <= set(a)
    return lumi_b200.lib().lumi_k_dequant_rows(*{**a, **k}.values())


def gemm(**k):
    a = dict(a=P, lda=64, a_scale=P, w=P, ldw=64, w_scale=P, bias=0, d=P, d_dtype=0, ldd=64, M=0, N=64, K=64, accumulate=0, status=0, stream=0)
    assert set(k) <= set(a)
    return lumi_b200.lib().lumi_k_gemm_i8(*{**a, **k}.values())


@pytest.mark.parametrize("k", [
    dict(x=0), dict(q=0), dict(scale=0), dict(x_dtype=2), dict(x_dtype=-1), dict(o_dtype=2), dict(rows=-1), dict(width=0), dict(width=-4), dict(width=65),
    dict(ldx=60), dict(ldx=66, width=60), dict(ldx=68, x_dtype=1), dict(ldo=60), dict(ldo=66), dict(ldo=68, o_dtype=1), dict(ldq=48), dict(ldq=72),
    dict(x=P + 4), dict(o=P + 8), dict(w=P + 4), dict(q=P + 8), dict(scale=P + 2), dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf"))])
def test_norm_refuses(k):
    assert norm(**k) == INVALID


@pytest.mark.parametrize("k", [
    dict(gu=0), dict(q=0), dict(scale=0), dict(dtype=2), dict(act=2), dict(act=-1), dict(rows=-1), dict(width=0), dict(up=60), dict(up=66, ld=136),
    dict(up=68, ld=136, dtype=1), dict(up=68), dict(ld=64, up=64), dict(ld=130), dict(ld=132, dtype=1), dict(ldq=48), dict(ldq=72), dict(gu=P + 4), dict(q=P + 8),
    dict(scale=P + 1), dict(up=2 ** 31 - 8)])
def test_gate_refuses(k):
    assert gate(**k) == INVALID


@pytest.mark.parametrize("k", [
    dict(q=0), dict(scale=0), dict(y=0), dict(y_dtype=2), dict(rows=-1), dict(width=0), dict(ldq=48), dict(ldq=72), dict(ldy=60),
    dict(q=P + 8), dict(scale=P + 2), dict(y=P + 2), dict(y=P + 1, y_dtype=1)])
def test_dequant_refuses(k):
    assert dequant(**k) == INVALID


@pytest.mark.parametrize("k,want", [
    (dict(a=0), INVALID), (dict(a_scale=0), INVALID), (dict(w=0), INVALID), (dict(w_scale=0), INVALID), (dict(d=0), INVALID), (dict(d_dtype=2), INVALID),
    (dict(M=-1), INVALID), (dict(N=-1), INVALID), (dict(K=0), INVALID), (dict(lda=48), INVALID), (dict(lda=72), INVALID), (dict(ldw=48), INVALID),
    (dict(ldw=72), INVALID), (dict(ldd=63), INVALID), (dict(a=P + 8), INVALID), (dict(w=P + 8), INVALID), (dict(a_scale=P + 2), INVALID),
    (dict(w_scale=P + 2), INVALID), (dict(bias=P + 2), INVALID), (dict(status=P + 2), INVALID), (dict(d=P + 2), INVALID), (dict(d=P + 1, d_dtype=1), INVALID),
    (dict(K=131072, lda=131072, ldw=131072), UNSUPPORTED), (dict(M=2 ** 30 + 1), UNSUPPORTED), (dict(N=2 ** 30 + 1, ldd=2 ** 30 + 1), UNSUPPORTED)])
def test_gemm_refuses(k, want):
    assert gemm(**k) == want


def test_rows_that_are_too_long():
    n = 2 ** 30 + 16
    assert norm(width=n, ldx=n, ldo=n, ldq=n) == UNSUPPORTED
    assert gate(width=n, up=n, ld=2 ** 31 - 64, ldq=n) == INVALID                  # two of them do not fit in a row


def test_nothing_to_do():
    assert norm() == 0 and norm(o=0, w=0, eps=0.0, ldo=0, o_dtype=9) == 0 and gate() == 0 and dequant() == 0
    assert gemm() == 0 and gemm(M=5, N=0, ldd=0) == 0 and gemm(K=131071, lda=131072, ldw=131072) == 0 and gemm(d=P + 2, d_dtype=1) == 0


def test_memory_that_is_not_the_devices_is_refused():
    """Host memory (or, without a device, any): refused, and nothing is launched."""
    import numpy as np
    x = np.zeros(4096, dtype=np.float32)
    p = (x.ctypes.data + 15) // 16 * 16
    k = dict(rows=1, x=p, o=0, w=p, q=p, scale=p)
    assert norm(**k) in (INVALID, CUDA)
    assert gate(rows=1, gu=p, q=p, scale=p) in (INVALID, CUDA)
    assert dequant(rows=1, q=p, scale=p, y=p) in (INVALID, CUDA)
    assert gemm(M=1, a=p, a_scale=p, w=p, w_scale=p, d=p) in (INVALID, CUDA)
    assert len(lumi_b200.lib().lumi_last_error()) > 0
