"""What the operators on rows of 8-bit integers are measured on: the norm and the gate that write such rows (`norm_quant`, `gate_quant`), and the product that
multiplies them (`gemm_i8`).

A row of numbers t is held as integers q in [-127, 127] and one fp32 scale s: m = max(max |t|, 2^-100), s = m / 127, q = t * 127 / m rounded to the nearest
integer, ties to even.  A case is a dict of plain values, `run` one pass: in plain torch where `own` is false, through the library where it is true."""
import torch

own = False

EPS = 1e-5
LEAST = 2.0 ** -100
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # the norm in front of a projection: one sequence's decode step; a batch of steps with a bf16 stream; a long prompt's rows
        dict(name="norm 1 x 1024", op="norm_quant", rows=1, width=1024, x="f32", o="f32", norm=True),
        dict(name="norm 64 x 2048 bf16", op="norm_quant", rows=64, width=2048, x="bf16", o="bf16", norm=True),
        dict(name="norm 32768 x 1024", op="norm_quant", rows=32768, width=1024, x="f32", o="f32", norm=True),
        # a projection's weights on their way into 8 bits, once per model: rows are output channels
        dict(name="weights 7360 x 1024 bf16", op="norm_quant", rows=7360, width=1024, x="bf16", o="none", norm=False),
        # the gate between the two products of a feed-forward: a few sequences' step; a long prompt
        dict(name="gate 8 x 2816", op="gate_quant", rows=8, width=2816, x="f32", act="sigmoid"),
        dict(name="gate 32768 x 2816 bf16", op="gate_quant", rows=32768, width=2816, x="bf16", act="silu"),
        # products: the input projection of one sequence's step
        dict(name="gemm 1 x 7360 x 1024", op="gemm_i8", M=1, N=7360, K=1024, d="f32", bias=False, add=False),
        # a feed-forward's second product into the residual stream, 16 sequences
        dict(name="gemm 16 x 1024 x 2816 add", op="gemm_i8", M=16, N=1024, K=2816, d="f32", bias=False, add=True),
        # no size a multiple of anything
        dict(name="gemm 203 x 2053 x 1111", op="gemm_i8", M=203, N=2053, K=1111, d="bf16", bias=True, add=False),
        # a step of 512 sequences
        dict(name="gemm 512 x 5632 x 2048", op="gemm_i8", M=512, N=5632, K=2048, d="bf16", bias=False, add=False),
        # prompts: the input projection, and a wide model's second product into its fp32 stream
        dict(name="gemm 4096 x 7360 x 1024", op="gemm_i8", M=4096, N=7360, K=1024, d="bf16", bias=False, add=False),
        dict(name="gemm 8192 x 2048 x 8448 add", op="gemm_i8", M=8192, N=2048, K=8448, d="f32", bias=False, add=True),
    ]


def _size(rng, low, high):
    """Spread over the logarithm; one in three as it falls, the others rounded to a multiple of 16 where that leaves something."""
    n = int(round(low * (high / low) ** rng.random()))
    if rng.random() < 2 / 3 and n > 16:
        n = (n + 8) // 16 * 16
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(["norm_quant", "gate_quant", "gemm_i8", "gemm_i8"])
    if op == "gemm_i8":
        while True:
            c = dict(op=op, M=_size(rng, 1, 16384), N=_size(rng, 8, 16384), K=_size(rng, 16, 16384), d=rng.choice(["f32", "bf16"]),
                     bias=rng.random() < 0.5, add=rng.random() < 0.5)
            if c["M"] * c["N"] * c["K"] <= 8192 * 2048 * 8448 and c["M"] * c["N"] <= 1 << 26:
                return c
    while True:
        rows, width = _size(rng, 1, 32768), _size(rng, 16, 16384)
        if rows * width <= 32768 * 1024:
            break
    x = rng.choice(["f32", "bf16"])
    if op == "gate_quant":
        return dict(op=op, rows=rows, width=width, x=x, act=rng.choice(["sigmoid", "silu"]))
    return dict(op=op, rows=rows, width=width, x=x, o=rng.choice(["none", "f32", "bf16"]), norm=rng.random() < 0.75)


def _up(n, k):
    return (n + k - 1) // k * k


def _normal(gen, rows, width, ld, dtype, factor=None):
    """Rows of `width` normal numbers in a buffer of rows of `ld`: the view of the numbers."""
    t = torch.randn(rows, width, generator=gen, device="cuda", dtype=torch.float32)
    if factor is not None:
        t *= factor
    buf = torch.zeros(rows, ld, device="cuda", dtype=dtype)
    buf[:, :width] = t
    return buf[:, :width]


def _codes(gen, rows, width):
    """8-bit rows as a quantiser leaves them: bell-shaped, the largest at 127 now and then."""
    t = torch.randn(rows, width, generator=gen, device="cuda", dtype=torch.float32)
    buf = torch.zeros(rows, _up(width, 16), device="cuda", dtype=torch.int8)
    buf[:, :width] = (t * 32).round_().clamp_(-127, 127)
    return buf[:, :width]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "gemm_i8":
        M, N, K = case["M"], case["N"], case["K"]
        s["a"], s["w"] = _codes(gen, M, K), _codes(gen, N, K)
        s["a_scale"] = torch.rand(M, generator=gen, device="cuda") * 0.02 + 0.005
        s["w_scale"] = torch.rand(N, generator=gen, device="cuda") * 1e-3 + 5e-4
        s["b"] = torch.randn(N, generator=gen, device="cuda") if case["bias"] else None
        s["out"] = _normal(gen, M, N, N, TYPES[case["d"]]) if case["add"] else torch.zeros(M, N, device="cuda", dtype=TYPES[case["d"]])
        return s
    rows, width = case["rows"], case["width"]
    s["q"] = torch.zeros(rows, _up(width, 16), device="cuda", dtype=torch.int8)[:, :width]
    s["scale"] = torch.zeros(rows, device="cuda")
    s["y"] = torch.zeros(rows, width, device="cuda", dtype=torch.bfloat16)
    if case["op"] == "gate_quant":
        s["up"] = _up(width, 16)
        s["gu"] = _normal(gen, rows, 2 * s["up"], 2 * s["up"], TYPES[case["x"]])
        return s
    # a few channels of a residual stream are much larger than the others
    factor = torch.where(torch.rand(width, generator=gen, device="cuda") < 0.01, 8.0, 1.0)
    s["v"] = _normal(gen, rows, width, _up(width, 16), TYPES[case["x"]], factor)
    s["add"] = _normal(gen, rows, width, _up(width, 16), TYPES[case["o"]], 0.25 * factor) if case["o"] != "none" else None
    s["w"] = 1 + 0.1 * torch.randn(width, generator=gen, device="cuda") if case["norm"] else None
    return s


def _quantised(t, factor=None):
    """Plain form: (values the 8-bit integers stand for, scales) of rows t, all times `factor` of the row."""
    m = t.abs().amax(dim=1, keepdim=True).clamp(min=LEAST)
    q = torch.round(t * (127 / m))
    scale = m / 127 if factor is None else m / 127 * factor
    return (q * scale).to(torch.bfloat16), scale[:, 0]


def _plain(s):
    if s["op"] == "gemm_i8":
        d = torch.matmul(s["a"].float(), s["w"].float().t()) * s["a_scale"][:, None] * s["w_scale"]
        if s["b"] is not None:
            d = d + s["b"]
        if s["add"]:
            d = d + s["out"].float()
        s["out"].copy_(d)
        return s["out"]
    if s["op"] == "gate_quant":
        g, u = s["gu"][:, :s["width"]].float(), s["gu"][:, s["up"]:s["up"] + s["width"]].float()
        t = 1 / (1 + torch.exp(-g))
        if s["act"] == "silu":
            t = g * t
        y, scale = _quantised(t * u)
        return {"y": y, "scale": scale}
    if s["add"] is not None:
        s["v"].copy_(s["v"].float() + s["add"].float())
    t, factor = s["v"].float(), None
    if s["w"] is not None:
        factor = 1 / torch.sqrt((t * t).mean(dim=1, keepdim=True) + EPS)
        t = t * s["w"]
    y, scale = _quantised(t, factor)
    return {"y": y, "scale": scale, "x": s["v"]}


def _dtype(t):
    return 1 if t.dtype == torch.bfloat16 else 0


def _library(s):
    import lumi_b200
    lib, check = lumi_b200.lib(), lumi_b200.api.check
    stream = torch.cuda.current_stream().cuda_stream
    if s["op"] == "gemm_i8":
        a, w, b, d = s["a"], s["w"], s["b"], s["out"]
        check(lib.lumi_k_gemm_i8(a.data_ptr(), a.stride(0), s["a_scale"].data_ptr(), w.data_ptr(), w.stride(0), s["w_scale"].data_ptr(),
                                 0 if b is None else b.data_ptr(), d.data_ptr(), _dtype(d), d.stride(0), s["M"], s["N"], s["K"], int(s["add"]), 0, stream))
        return d
    q, scale, y = s["q"], s["scale"], s["y"]
    if s["op"] == "gate_quant":
        gu = s["gu"]
        check(lib.lumi_k_gate_quant(gu.data_ptr(), _dtype(gu), gu.stride(0), s["up"], 1 if s["act"] == "silu" else 0, q.data_ptr(), q.stride(0),
                                    scale.data_ptr(), s["rows"], s["width"], stream))
        check(lib.lumi_k_dequant_rows(q.data_ptr(), q.stride(0), scale.data_ptr(), y.data_ptr(), 1, y.stride(0), s["rows"], s["width"], stream))
        return {"y": y, "scale": scale}
    v, o, w = s["v"], s["add"], s["w"]
    check(lib.lumi_k_norm_quant(v.data_ptr(), _dtype(v), v.stride(0), 0 if o is None else o.data_ptr(), 0 if o is None else _dtype(o),
                                0 if o is None else o.stride(0), 0 if w is None else w.data_ptr(), q.data_ptr(), q.stride(0), scale.data_ptr(),
                                s["rows"], s["width"], EPS, stream))
    check(lib.lumi_k_dequant_rows(q.data_ptr(), q.stride(0), scale.data_ptr(), y.data_ptr(), 1, y.stride(0), s["rows"], s["width"], stream))
    return {"y": y, "scale": scale, "x": v}


def run(state):
    return _library(state) if own else _plain(state)


def exact(case, seed):
    """The definitions in 64 bits.  Sums of products of 8-bit integers are whole numbers below 2^53, which 64-bit products hold exactly."""
    s = prepare(case, seed)
    if case["op"] == "gemm_i8":
        total = s["a"].double() @ s["w"].double().t()
        total *= s["a_scale"].double().outer(s["w_scale"].double())
        if s["b"] is not None:
            total += s["b"].double()
        if case["add"]:
            total += s["out"].double()
        return total
    if case["op"] == "gate_quant":
        both = s["gu"].double().reshape(case["rows"], 2, s["up"])[:, :, :case["width"]]
        gate, up = both[:, 0], both[:, 1]
        z = torch.sigmoid(gate) * up * (gate if case["act"] == "silu" else 1)
        x = None
    else:
        z = s["v"].double()
        if s["add"] is not None:
            z = z + s["add"].double()
        x = z
        if case["x"] == "bf16":
            z = z.to(torch.float32).to(torch.bfloat16).double()      # the stored stream is what the norm sees
    largest = z.abs()
    if case["op"] == "norm_quant" and case["norm"]:
        norm = (z.pow(2).sum(1, keepdim=True) / case["width"] + EPS).rsqrt()
        z = z * s["w"].double()
        largest = z.abs()
    else:
        norm = torch.ones(case["rows"], 1, device="cuda", dtype=torch.float64)
    step = largest.max(1, keepdim=True).values.clamp(min=LEAST) / 127
    y = torch.round(z / step) * step * norm
    out = {"y": y, "scale": (step * norm).squeeze(1)}
    return out if x is None else {**out, "x": x}


def work(case):
    """Every input read once, every output written once."""
    if case["op"] == "gemm_i8":
        M, N, K, e = case["M"], case["N"], case["K"], TYPES[case["d"]].itemsize
        return {"bytes": M * K + N * K + M * N * e * (2 if case["add"] else 1) + 4 * (M + N * (2 if case["bias"] else 1)), "flops": 2 * M * N * K}
    n, e = case["rows"] * case["width"], TYPES[case["x"]].itemsize
    if case["op"] == "gate_quant":
        return {"bytes": n * (2 * e + 1) + 4 * case["rows"], "flops": 12 * n}
    o = 0 if case["o"] == "none" else TYPES[case["o"]].itemsize + e      # read, and the sum written
    return {"bytes": n * (e + o + 1) + 4 * case["rows"] + (4 * case["width"] if case["norm"] else 0), "flops": 6 * n}
