"""CPU: what the calls on a cache in 4 bits and the block norm refuse, before a device is touched; the layout that the other tests take their numbers from.  Addresses are made up."""
import ctypes as C

import numpy as np
import pytest

import kv4_reference as ref
import lumi_b200

INVALID, UNSUPPORTED = -1, -10
P = 1 << 20      # an address on a 16-byte boundary


def call(name, defaults, k):
    assert set(k) <= set(defaults)
    return getattr(lumi_b200.lib(), name)(*{**defaults, **k}.values())


def plan(**k):
    return call("lumi_k_page_plan", dict(tokens=P, len=P, nseq=4, table=P, width=4, free=P, n_pages=16, pool=P, pool_after=P, tokens_after=P, row_start=P, pos=P, slot=P, rows=8,
                                         stream=0), k)


def append(**k):
    return call("lumi_k_kv4_append", dict(k=P, ldk=128, v=P, ldv=128, dtype=0, slot=P, kv=P, n_pages=4, kv_heads=2, dk=64, dv=64, rows=0, stream=0), k)


def read(**k):
    return call("lumi_k_kv4_read", dict(kv=P, n_pages=4, slot=P, k=P, ldk=128, v=P, ldv=128, dtype=0, kv_heads=2, dk=64, dv=64, rows=0, stream=0), k)


def attention(**k):
    return call("lumi_k_kv4_attention", dict(q=P, ldq=256, dtype=0, kv=P, n_pages=4, table=P, width=4, row_start=P, tokens=P, y=P, ldy=256, heads=4, kv_heads=2, dk=64, dv=64, window=0,
                                             scale=0.125, sink=0, nseq=1, rows=0, max_new=1, work=P, work_bytes=1 << 30, status=0, stream=0), k)


def block_norm(**k):
    return call("lumi_k_block_norm", dict(x=P, x_dtype=0, ldx=64, o=P, o_dtype=0, ldo=64, w_post=P, gate=P, ldg=64, scale=1.0, w_pre=P, y=P, y_dtype=0, ldy=64, rows=0, width=64,
                                          eps=1e-5, stream=0), k)


@pytest.mark.parametrize("k,want", [(dict([(n, 0)]), INVALID) for n in ("tokens", "len", "table", "free", "pool", "pool_after", "tokens_after", "row_start", "pos", "slot")] + [
    (dict(nseq=-1), INVALID), (dict(width=0), INVALID), (dict(n_pages=0), INVALID), (dict(rows=-1), INVALID), (dict(tokens=P + 2), INVALID), (dict(slot=P + 1), INVALID),
    (dict(nseq=8193), UNSUPPORTED), (dict(n_pages=1 << 25), UNSUPPORTED), (dict(width=1 << 25), UNSUPPORTED)])
def test_plan_refuses(k, want):
    assert plan(**k) == want


ROWS = [(dict(k=0), INVALID), (dict(v=0), INVALID), (dict(slot=0), INVALID), (dict(kv=0), INVALID), (dict(dtype=2), INVALID), (dict(rows=-1), INVALID), (dict(n_pages=0), INVALID),
        (dict(kv_heads=0), INVALID), (dict(dk=0), INVALID), (dict(dv=-1), INVALID), (dict(ldk=127), INVALID), (dict(ldv=64), INVALID), (dict(k=P + 2), INVALID), (dict(v=P + 1, dtype=1), INVALID),
        (dict(slot=P + 2), INVALID), (dict(kv=P + 8), INVALID), (dict(dk=257, ldk=1024), UNSUPPORTED), (dict(dv=300, ldv=1024), UNSUPPORTED), (dict(n_pages=1 << 25), UNSUPPORTED)]


@pytest.mark.parametrize("k,want", ROWS)
def test_append_and_read_refuse(k, want):
    assert append(**k) == want and read(**k) == want


def test_calls_without_rows_do_nothing():
    assert append() == 0 and read() == 0 and block_norm() == 0 and attention() == 0 and attention(rows=4, nseq=0) == 0 and attention(rows=4, max_new=0) == 0


@pytest.mark.parametrize("k,want", [(dict([(n, 0)]), INVALID) for n in ("q", "kv", "table", "row_start", "tokens", "y", "work")] + [
    (dict(dtype=2), INVALID), (dict(n_pages=0), INVALID), (dict(width=0), INVALID), (dict(heads=0), INVALID), (dict(heads=3), INVALID), (dict(kv_heads=0), INVALID), (dict(dk=0), INVALID),
    (dict(dv=0), INVALID), (dict(window=-1), INVALID), (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID), (dict(nseq=-1), INVALID), (dict(rows=-1), INVALID),
    (dict(max_new=-1), INVALID), (dict(ldq=255), INVALID), (dict(ldy=255), INVALID), (dict(kv=P + 8), INVALID), (dict(work=P + 8), INVALID), (dict(table=P + 2), INVALID),
    (dict(tokens=P + 1), INVALID), (dict(status=P + 2), INVALID), (dict(q=P + 2), INVALID), (dict(y=P + 1, dtype=1), INVALID), (dict(work_bytes=1024), INVALID),
    (dict(dk=257, ldq=2000), UNSUPPORTED), (dict(dv=257, ldy=2000), UNSUPPORTED), (dict(n_pages=1 << 25), UNSUPPORTED), (dict(rows=(1 << 24) + 1), UNSUPPORTED),
    (dict(rows=1 << 24, max_new=1 << 24, heads=128, kv_heads=1, dk=1, dv=1), UNSUPPORTED), (dict(heads=65536, kv_heads=1, dk=1, dv=1, ldq=65536, ldy=65536), UNSUPPORTED)])
def test_attention_refuses(k, want):
    assert attention(**k) == want


def test_the_hook_refuses_what_the_call_does():
    base = dict(q=P, ldq=256, dtype=0, kv=P, n_pages=4, table=P, width=4, row_start=P, tokens=P, y=P, ldy=256, heads=4, kv_heads=2, dk=64, dv=64, window=0, scale=0.125, sink=0, nseq=1, rows=4,
                max_new=1, work=P, work_bytes=1 << 30, status=P, wait_ns=1000, skip=-1)
    for k, want in ((dict(status=0), INVALID), (dict(wait_ns=0), INVALID), (dict(q=0), INVALID), (dict(heads=3), INVALID), (dict(dk=257, ldq=2000), UNSUPPORTED)):
        assert call("lumi_debug_kv4_attention_wait_timeout", base, k) == want


def test_work_areas():
    n = C.c_int64()
    get = lambda *a: lumi_b200.lib().lumi_k_kv4_attention_work_bytes(*a, C.byref(n))
    assert get(64, 8, 128, 128) == 0 and n.value >= 320 * 256 * (2 + 128) * 4 + 4096
    assert get(0, 1, 64, 64) == INVALID and get(3, 2, 64, 64) == INVALID and get(4, 2, 0, 64) == INVALID and lumi_b200.lib().lumi_k_kv4_attention_work_bytes(4, 2, 64, 64, None) == INVALID
    assert get(4, 2, 257, 64) == UNSUPPORTED and get(4, 2, 64, 300) == UNSUPPORTED and get(65536, 1, 64, 64) == UNSUPPORTED


def test_more_groups_than_a_launch_takes():
    assert append(kv_heads=65535, dk=256, dv=256, ldk=1 << 24, ldv=1 << 24) == UNSUPPORTED and append(kv_heads=65535, dk=128, dv=128, ldk=1 << 24, ldv=1 << 24) == 0


@pytest.mark.parametrize("k,want", [
    (dict(x=0), INVALID), (dict(o=0), INVALID), (dict(w_pre=0), INVALID), (dict(x_dtype=2), INVALID), (dict(o_dtype=-1), INVALID), (dict(y_dtype=3), INVALID), (dict(rows=-1), INVALID),
    (dict(width=0), INVALID), (dict(ldx=60), INVALID), (dict(ldo=60), INVALID), (dict(ldg=60), INVALID), (dict(ldy=60), INVALID), (dict(ldx=66), INVALID), (dict(ldx=68, x_dtype=1), INVALID),
    (dict(x=P + 8), INVALID), (dict(o=P + 4), INVALID), (dict(gate=P + 4), INVALID), (dict(y=P + 8), INVALID), (dict(w_post=P + 4), INVALID), (dict(w_pre=P + 8), INVALID),
    (dict(eps=0.0), INVALID), (dict(eps=float("nan")), INVALID), (dict(width=32769, ldx=32776, ldo=32776, ldg=0, ldy=32776), UNSUPPORTED)])
def test_block_norm_refuses(k, want):
    assert block_norm(**k) == want


def test_block_norm_takes_less():
    assert block_norm(w_post=0, gate=0, y=0, w_pre=0, eps=0.0) == 0 and block_norm(ldg=0) == 0


@pytest.mark.parametrize("heads,dk,dv", [(1, 1, 1), (8, 128, 128), (4, 64, 64), (3, 80, 100), (2, 256, 33)])
def test_page_bytes(heads, dk, dv):
    n = C.c_int64()
    assert lumi_b200.lib().lumi_k_kv4_page_bytes(heads, dk, dv, C.byref(n)) == 0 and n.value == heads * ref.block_bytes(dk, dv) and n.value % 16 == 0
    assert lumi_b200.lib().lumi_k_kv4_page_bytes(heads, 257, dv, C.byref(n)) == UNSUPPORTED and lumi_b200.lib().lumi_k_kv4_page_bytes(0, dk, dv, C.byref(n)) == INVALID


def test_work_bytes():
    n = C.c_int64()
    lib = lumi_b200.lib()
    assert lib.lumi_k_kv4_attention_work_bytes(64, 8, 256, 256, C.byref(n)) == 0 and 0 < n.value <= 64 << 20
    assert lib.lumi_k_kv4_attention_work_bytes(3, 2, 64, 64, C.byref(n)) == INVALID and lib.lumi_k_kv4_attention_work_bytes(4, 2, 64, 64, None) == INVALID


def test_reference_round_trip():
    """The layout of the reference: what is written at a slot is what is read there, and half a step off at most."""
    rng = np.random.default_rng(0)
    for dk, dv in ((64, 64), (33, 100), (1, 7)):
        cache = rng.integers(0, 256, (3, 2, ref.block_bytes(dk, dv)), dtype=np.uint8)
        slots = [5, 64, 63, 130]
        k, v = rng.standard_normal((4, 2, dk)).astype(np.float32), rng.standard_normal((4, 2, dv)).astype(np.float32)
        for i, s in enumerate(slots):
            for h in range(2):
                ref.write(cache, s, h, k[i, h], v[i, h])
        for got, t in zip(ref.read(cache, slots, dk, dv), (k, v)):
            codes, scales = ref.quantise(t)
            assert np.array_equal(got, ref.values(codes, scales)) and codes.min() >= 1 and codes.max() <= 15
            assert (np.abs(got - t) <= np.repeat(scales, 32, -1)[..., :t.shape[-1]] * (0.5 + 2 ** -20)).all()
