"""GPU: rows as 8-bit integers with a scale (lumi_k_norm_quant, lumi_k_gate_quant, lumi_k_dequant_rows) against the definition in 64 bits.

Tolerances, from the arithmetic (u = 2^-24, a rounding to fp32):
* x + o: one rounding to fp32 (u), and for a bf16 stream one more (2^-8): compared with the same two roundings, which torch makes as well: equal.
* scale without norm: m is exact, m / 127 one rounding: u.  With norm: the products x w round once (u), the quotient and the product with r once each, the sum
  of squares over n elements is a tree of at most 64 serial additions per thread and 10 levels behind (each 1 u of a sum of positive terms, halved by the
  root), its quotient, the sum with eps, root and reciprocal 1 u each: (74 / 2 + 8) u < 2^-18.
* the gate: exp and the quotient are good to a few 2^-22 relative, times the size of the argument where the gate is far below zero: 2^-18 of |t| for
  |gate| < 16, which is where the tests draw.
* integers: t * 127 / m is off by at most 127 * (e + 2 u), e the relative error of t against m: an integer may differ from rint of the exact quotient only where that lies
  that near a half.  So |q s - t| <= s (1 / 2 + that)."""
import itertools

import pytest
import torch

import lumi_b200

pytestmark = pytest.mark.gpu
LEAST = 2.0 ** -100
SCALE_TOL = 2.0 ** -18
EPS = 1e-5


def call(name, *args):
    lumi_b200.api.check(getattr(lumi_b200.lib(), name)(*args))


def code(t):
    return 1 if t.dtype == torch.bfloat16 else 0


def rows_of(t, ld, dtype, fill=7.0):
    """t in rows of ld elements; what lies between the rows holds `fill`."""
    buf = torch.full((t.shape[0], ld), fill, device="cuda", dtype=dtype)
    buf[:, :t.shape[1]] = t
    return buf


def norm(x, o, w, width, ldq, eps=EPS, stream=0):
    q = torch.full((x.shape[0], ldq), 99, device="cuda", dtype=torch.int8)
    s = torch.full((x.shape[0] + 1,), -1.0, device="cuda")
    call("lumi_k_norm_quant", x.data_ptr(), code(x), x.stride(0), 0 if o is None else o.data_ptr(), 0 if o is None else code(o),
         0 if o is None else o.stride(0), 0 if w is None else w.data_ptr(), q.data_ptr(), ldq, s.data_ptr(), x.shape[0], width, eps, stream)
    torch.cuda.synchronize()
    assert float(s[-1]) == -1.0 and bool((q[:, width:] == 99).all())      # what lies behind is left alone
    return q[:, :width].double(), s[:-1].double()


def check(q, s, t, factor, tol):
    """q and s against rows t (64 bits), all times factor [rows, 1]."""
    m = t.abs().amax(1).clamp(min=LEAST)
    want = m / 127 * factor[:, 0]
    assert float(((s - want).abs() / want).max()) <= SCALE_TOL
    assert float(q.abs().max()) <= 127
    steps = t / (m[:, None] / 127)
    assert float((q - steps).abs().max()) <= 0.5 + 127 * (tol + 2.0 ** -22)
    assert bool((q.abs().amax(1)[m > LEAST] == 127).all())


WIDTHS = [1, 3, 8, 31, 100, 255, 256, 1000, 1024, 1031, 2048, 2816, 4100, 7360, 8192, 8200, 16384, 20001]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("x_dtype,o_dtype", list(itertools.product([torch.float32, torch.bfloat16], [None, torch.float32, torch.bfloat16])))
def test_norm(width, x_dtype, o_dtype):
    g = torch.Generator(device="cuda").manual_seed(width)
    for rows, pad, with_norm in ((1, 0, True), (5, 16, True), (5, 0, False), (613, 0, True)):
        if rows * width > 3_000_000:
            continue
        ld = (width + 15) // 16 * 16 + pad
        x0 = torch.randn(rows, width, generator=g, device="cuda") * 3
        x = rows_of(x0, ld, x_dtype)
        o = None if o_dtype is None else rows_of(torch.randn(rows, width, generator=g, device="cuda"), ld + 8, o_dtype, float("nan"))
        w = torch.randn(width, generator=g, device="cuda") if with_norm else None
        stream = x[:, :width].clone()
        if o is not None:
            stream = (stream.float() + o[:, :width].float()).to(x_dtype)
        q, s = norm(x, o, w, width, ld)
        assert torch.equal(x[:, :width], stream) and bool((x[:, width:] == 7).all())
        t = stream.double()
        factor = torch.ones(rows, 1, device="cuda", dtype=torch.float64)
        if with_norm:
            factor = 1 / torch.sqrt((t * t).mean(1, keepdim=True) + EPS)
            t = t * w.double()
        check(q, s, t, factor, 2.0 ** -24)


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", [0, 1])
def test_gate(width, dtype, act):
    g = torch.Generator(device="cuda").manual_seed(width + act)
    for rows, pad in ((1, 0), (7, 16), (641, 0)):
        if rows * width > 3_000_000:
            continue
        up = (width + 15) // 16 * 16 + pad
        gate = (torch.randn(rows, width, generator=g, device="cuda") * 4).clamp(-15.9, 15.9)
        ups = torch.randn(rows, width, generator=g, device="cuda")
        gu = rows_of(gate, 2 * up + pad, dtype, float("nan"))
        gu[:, up:up + width] = ups
        z, u = gu[:, :width].double(), gu[:, up:up + width].double()
        ldq = (width + 15) // 16 * 16
        q = torch.full((rows, ldq), 99, device="cuda", dtype=torch.int8)
        s = torch.full((rows + 1,), -1.0, device="cuda")
        call("lumi_k_gate_quant", gu.data_ptr(), code(gu), gu.stride(0), up, act, q.data_ptr(), ldq, s.data_ptr(), rows, width, 0)
        torch.cuda.synchronize()
        assert float(s[-1]) == -1.0 and bool((q[:, width:] == 99).all())
        t = torch.sigmoid(z) * u * (z if act else 1)
        check(q[:, :width].double(), s[:-1].double(), t, torch.ones(rows, 1, device="cuda", dtype=torch.float64), 2.0 ** -18)


@pytest.mark.parametrize("width", [5, 1024, 8192, 20001])
def test_rows_of_zeros_small_and_large_numbers_and_of_none(width):
    """Zeros give zeros; rows near the ends of fp32 keep their integers; an infinity or a NaN in a row gives NaN for that row alone."""
    ld = (width + 15) // 16 * 16
    g = torch.Generator(device="cuda").manual_seed(1)
    base = torch.randn(8, width, generator=g, device="cuda")
    base[0] = 0
    base[1] *= 1e-29
    base[2] *= 1e25
    base[3, width // 2] = float("inf")
    base[4, width - 1] = float("nan")
    base[5, 0] = float("-inf")
    base[6] = 0
    base[6, width - 1] = -2.0                             # one number alone
    x = rows_of(base, ld, torch.float32)
    ones = torch.ones(width, device="cuda")
    for w in (None, ones):
        q, s = norm(x.clone(), None, w, width, ld)
        assert bool(torch.isnan(s[3:6]).all()) and bool((q[3:6] == 0).all())
        keep = [0, 1, 2, 6, 7]
        t = base[keep].double()
        factor = torch.ones(5, 1, device="cuda", dtype=torch.float64)
        if w is not None:
            factor = 1 / torch.sqrt((t * t).mean(1, keepdim=True) + EPS)
        m = t.abs().amax(1).clamp(min=LEAST)
        assert float(((s[keep] - m / 127 * factor[:, 0]).abs() / (m / 127 * factor[:, 0])).max()) <= SCALE_TOL
        assert float((q[keep] - t / (m[:, None] / 127)).abs().max()) <= 0.5 + 127 * 2.0 ** -21
        assert bool((q[0] == 0).all())
    tiny = rows_of(torch.full((1, width), 1e-38, device="cuda"), ld, torch.float32)       # below 2^-100: held as zeros
    q, s = norm(tiny, None, None, width, ld)
    assert bool((q == 0).all()) and float(s[0]) == pytest.approx(LEAST / 127)


def test_sums_of_squares_beyond_fp32():
    """Squares that overflow, and squares that vanish beside a small eps, are taken again with the row scaled."""
    width = 1024
    g = torch.Generator(device="cuda").manual_seed(2)
    for size, eps in ((1e30, 1e-5), (1e20, 1e-5), (1e-25, 1e-37), (1e-21, 1e-30)):
        for wide in (width, 20000):
            t = torch.randn(3, wide, generator=g, device="cuda") * size
            q, s = norm(rows_of(t, wide, torch.float32), None, torch.ones(wide, device="cuda"), wide, wide, eps)
            t = t.double()
            check(q, s, t, 1 / torch.sqrt((t * t).mean(1, keepdim=True) + float(torch.tensor(eps))), 2.0 ** -24)


def test_same_bits_alone_and_among_others_and_again():
    """A row's integers and scale do not depend on how many rows there are, nor on the run."""
    g = torch.Generator(device="cuda").manual_seed(3)
    for width in (96, 1024, 2048, 5632):
        x = torch.randn(1500, width, generator=g, device="cuda")
        w = torch.randn(width, generator=g, device="cuda")
        q, s = norm(x.clone(), None, w, width, width)
        q2, s2 = norm(x.clone(), None, w, width, width)
        assert torch.equal(q, q2) and torch.equal(s, s2)
        for r in (0, 777, 1499):
            q1, s1 = norm(x[r:r + 1].clone(), None, w, width, width)
            assert torch.equal(q1[0], q[r]) and torch.equal(s1[0], s[r])


def test_residual_onto_itself():
    """o may be x: the rows are doubled."""
    x = torch.randn(4, 1024, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    want = x * 2
    q, s = norm(x, x, None, 1024, 1024)
    assert torch.equal(x, want)
    check(q, s, want.double(), torch.ones(4, 1, device="cuda", dtype=torch.float64), 2.0 ** -24)


def test_offsets_past_31_bits():
    """Rows further than 2^31 elements from the first."""
    width, ld, rows = 64, 1 << 20, 2100
    x = torch.empty(rows * ld, device="cuda", dtype=torch.bfloat16)                  # 4.4 GB, 2.2e9 elements
    v = x.view(rows, ld)[:, :width]
    v.copy_(torch.randn(rows, width, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)))
    q = torch.empty(rows * ld, device="cuda", dtype=torch.int8)
    s = torch.empty(rows, device="cuda")
    call("lumi_k_norm_quant", x.data_ptr(), 1, ld, 0, 0, 0, 0, q.data_ptr(), ld, s.data_ptr(), rows, width, 0.0, 0)
    torch.cuda.synchronize()
    check(q.view(rows, ld)[:, :width].double(), s.double(), v.double(), torch.ones(rows, 1, device="cuda", dtype=torch.float64), 2.0 ** -24)


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_back(width, dtype):
    """One product in fp32, for bf16 rounded once more: torch's own is the same bits.  -128 is allowed; a NaN or infinite scale is its row's alone."""
    g = torch.Generator(device="cuda").manual_seed(width)
    for rows, pad in ((1, 0), (9, 16), (300, 0)):
        ld = (width + 15) // 16 * 16 + pad
        q = torch.randint(-128, 128, (rows, ld), generator=g, device="cuda", dtype=torch.int16).to(torch.int8)
        s = torch.randn(rows + 1, generator=g, device="cuda")
        if rows > 2:
            s[1], s[2] = float("nan"), float("inf")
        for ldy, shift in ((ld, 0), (width, 0), (width + 1, 1)):
            whole = torch.full((rows * ldy + 8,), 7.0, device="cuda", dtype=dtype)
            y = whole[shift:shift + rows * ldy].view(rows, ldy)
            call("lumi_k_dequant_rows", q.data_ptr(), ld, s.data_ptr(), y.data_ptr(), code(y), ldy, rows, width, 0)
            torch.cuda.synchronize()
            assert bool((y[:, width:] == 7).all()) and bool((whole[:shift] == 7).all()) and bool((whole[shift + rows * ldy:] == 7).all())
            assert torch.equal((q[:, :width].float() * s[:rows, None]).to(dtype).nan_to_num(nan=1e30), y[:, :width].nan_to_num(nan=1e30))


@pytest.mark.parametrize("width", [5, 260, 1001, 4100, 70001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_that_begin_on_16_bytes_and_no_more(width, dtype):
    """Bases 16 bytes behind a larger boundary, rows that are whole 16 bytes long and no more, operands that end where they do."""
    e = 128 // torch.finfo(dtype).bits
    ld, ldq, rows = (width + e - 1) // e * e, (width + 15) // 16 * 16, 3
    g = torch.Generator(device="cuda").manual_seed(width)

    def rows_at(ld, dtype, step):
        buf = torch.zeros(step + (rows - 1) * ld + width, device="cuda", dtype=dtype)      # the last row ends with its numbers
        return buf, buf[step:].as_strided((rows, width), (ld, 1))

    _, x = rows_at(ld, dtype, e)
    _, o = rows_at(ld, dtype, e)
    for t in (x, o):
        t.copy_(torch.randn(rows, width, generator=g, device="cuda"))
    w = torch.zeros(4 + width, device="cuda")[4:]
    w.copy_(torch.randn(width, generator=g, device="cuda"))
    whole, q = rows_at(ldq, torch.int8, 16)
    s = torch.zeros(rows + 1, device="cuda")[1:]
    want = (x.float() + o.float()).to(dtype)
    call("lumi_k_norm_quant", x.data_ptr(), code(x), ld, o.data_ptr(), code(o), ld, w.data_ptr(), q.data_ptr(), ldq, s.data_ptr(), rows, width, EPS, 0)
    torch.cuda.synchronize()
    assert torch.equal(x, want) and bool((whole[:16] == 0).all())
    t = want.double()
    check(q.double(), s.double(), t * w.double(), 1 / torch.sqrt((t * t).mean(1, keepdim=True) + EPS), 2.0 ** -24)
    up = ld
    buf = torch.zeros(e + (rows - 1) * 2 * up + up + width, device="cuda", dtype=dtype)
    gu = buf[e:]
    gate, ups = gu.as_strided((rows, width), (2 * up, 1)), gu[up:].as_strided((rows, width), (2 * up, 1))
    gate.copy_(x.clamp(-15, 15)), ups.copy_(o)
    call("lumi_k_gate_quant", gu.data_ptr(), code(gu), 2 * up, up, 1, q.data_ptr(), ldq, s.data_ptr(), rows, width, 0)
    torch.cuda.synchronize()
    z = gate.double()
    check(q.double(), s.double(), torch.sigmoid(z) * z * ups.double(), torch.ones(rows, 1, device="cuda", dtype=torch.float64), 2.0 ** -18)
    y = torch.zeros(rows * width + 1, device="cuda", dtype=dtype)[1:].view(rows, width)
    call("lumi_k_dequant_rows", q.data_ptr(), ldq, s.data_ptr(), y.data_ptr(), code(y), width, rows, width, 0)
    torch.cuda.synchronize()
    assert torch.equal(y, (q.float() * s[:, None]).to(dtype))


@pytest.mark.parametrize("width", [33, 256, 1000, 2048, 8192, 20001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_definitions_own_bits(width, dtype):
    """q = rint(t * (127 / m)), every operation in fp32, also of numbers that lie on halves of a step; and scales without a norm are m / 127.  The quotients are taken in 64
    bits and rounded, which is their fp32 rounding (53 >= 2 * 24 + 2); torch's own divisions by and of a number multiply by a reciprocal instead."""
    g = torch.Generator(device="cuda").manual_seed(width)
    x = torch.randn(40, width, generator=g, device="cuda")
    x[20:] = torch.randint(-508, 509, (20, width), generator=g, device="cuda") / 4          # quarters of steps, where the largest is 127
    x[20:, 0] = 127
    x[20:].clamp_(-127, 127)
    rows = rows_of(x, (width + 15) // 16 * 16, dtype)
    w = torch.randn(width, generator=g, device="cuda")
    for weights in (None, w):
        q, s = norm(rows.clone(), None, weights, width, (width + 15) // 16 * 16)
        t = rows[:, :width].float()
        if weights is not None:
            t = t * weights
        m = t.abs().amax(1, keepdim=True)
        assert torch.equal(q.float(), torch.round(t * (127 / m.double()).float()))
        if weights is None:
            assert torch.equal(s.float(), (m.double() / 127).float()[:, 0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [16, 704, 4096, 20000])
def test_gates_far_from_zero(dtype, width):
    """Gates at +-100, +-88, +-30 and, for the sigmoid, infinite ones: open or closed, and closed to zero.  (Below -16 the gate's relative error grows to |gate| 2^-23, of numbers
    under e^-16 of the row's largest: nothing beside half a step.)  An open silu of an infinity is an infinity: that row is NaN, and its neighbours are not."""
    g = torch.Generator(device="cuda").manual_seed(width)
    some = torch.tensor([-100.0, -88, -30, -17, 0, 17, 30, 88, 100, -1000], device="cuda")
    gate = some[torch.randint(0, 10, (4, width), generator=g, device="cuda")]
    ups = torch.randn(4, width, generator=g, device="cuda")
    gate[:, 0], ups[:, 0] = 100, 1
    for act in (0, 1):
        z = gate.clone()
        if act == 0:
            z[1, 1], z[2, 2] = float("-inf"), float("inf")
        else:
            z[2, 2] = float("inf")
            ups[2, 2] = 1
        gu = torch.cat([z, ups], 1).to(dtype).contiguous()
        q = torch.zeros(4, (width + 15) // 16 * 16, device="cuda", dtype=torch.int8)
        s = torch.zeros(4, device="cuda")
        call("lumi_k_gate_quant", gu.data_ptr(), code(gu), 2 * width, width, act, q.data_ptr(), q.stride(0), s.data_ptr(), 4, width, 0)
        torch.cuda.synchronize()
        zd, ud = gu[:, :width].double(), gu[:, width:].double()
        t = torch.sigmoid(zd) * ud * (zd if act else 1)
        keep = [0, 1, 2, 3] if act == 0 else [0, 1, 3]
        check(q[keep][:, :width].double(), s[keep].double(), t[keep], torch.ones(len(keep), 1, device="cuda", dtype=torch.float64), 2.0 ** -18)
        if act == 1:
            assert bool(torch.isnan(s[2])) and bool((q[2] == 0).all())
