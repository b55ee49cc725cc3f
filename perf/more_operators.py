"""What the operators around attention over a cache in 4 bits are measured on: page tables and slots made from the lengths of requests (`plan`), keys and values
into the cache and back (`append`), attention over it (`attend`), and the norms before and after a block with its gate and residual scale (`block_norm`).

The cache holds pages of 64 tokens; a page has a block per head of keys and values.  32 numbers t of a token and head are a group: m = max(max |t|, 2^-100), the scale s is m / 7
rounded up to bf16, and number t is held as n = 8 + rint(t / s) in 4 bits (fp32 quotient, ties to even): t is about (n - 8) s.  A block is keys' codes, keys' scales,
values' codes, values' scales; codes lie as [group][token][16 bytes], scales as [group][token] bf16.  Of a group's 16 bytes, number i of the values is nibble i; of the keys,
four words hold eight numbers each, number e of a word as nibble e / 2 + 4 (e % 2).

A case is a dict of plain values, `run` one pass: in plain torch where `own` is false, through the library where it is true."""
import math
import random

import torch

own = False

EPS = 1e-5
LEAST = 2.0 ** -100
PAGE = 64
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # a step of 256 sequences: one more token each; a scheduler's tick over 2048 slots: steps, prompts of up to 2048 tokens, requests that have ended
        dict(name="plan 256 steps", op="plan", nseq=256, most=1, pages=128),
        dict(name="plan 2048 mixed", op="plan", nseq=2048, most=2048, pages=128),
        # a step of 64 sequences into the cache; rows of prompts as the fp32 projections leave them
        dict(name="append 64 x 8 x 128 bf16", op="append", rows=64, kv_heads=8, dk=128, dv=128, type="bf16"),
        dict(name="append 65536 x 4 x 64", op="append", rows=65536, kv_heads=4, dk=64, dv=64, type="f32"),
        # one sequence's step in the hybrid's attention layer
        dict(name="step 1 of 4000, 16/4 x 64", op="attend", nseq=1, new=1, held=3999, even=True, heads=16, kv_heads=4, dk=64, dv=64, window=0, sink=False, type="f32"),
        # a batch of steps over contexts of very different lengths; a few long ones
        dict(name="steps 64 up to 8192, 32/8 x 128 bf16", op="attend", nseq=64, new=1, held=8191, even=False, heads=32, kv_heads=8, dk=128, dv=128, window=0, sink=False,
             type="bf16"),
        dict(name="steps 8 of 32000, 64/8 x 128 bf16", op="attend", nseq=8, new=1, held=31999, even=True, heads=64, kv_heads=8, dk=128, dv=128, window=0, sink=False, type="bf16"),
        # sliding windows with a softmax sink, a key head per query head, heads that are no power of two
        dict(name="steps 256 window 1024, 16/16 x 80 sink", op="attend", nseq=256, new=1, held=2500, even=False, heads=16, kv_heads=16, dk=80, dv=80, window=1024, sink=True,
             type="f32"),
        # prompts; a slice of a long prompt behind what is held already
        dict(name="prompts 8 x 2048, 16/4 x 64 bf16", op="attend", nseq=8, new=2048, held=0, even=True, heads=16, kv_heads=4, dk=64, dv=64, window=0, sink=False, type="bf16"),
        dict(name="slices 2 x 512 behind 16000, 32/8 x 128 bf16", op="attend", nseq=2, new=512, held=16000, even=True, heads=32, kv_heads=8, dk=128, dv=128, window=0, sink=False,
             type="bf16"),
        # the norms around a block: one sequence's step; a long prompt's rows
        dict(name="block norm 1 x 1024", op="block_norm", rows=1, width=1024, x="f32", o="f32", gate="none", y="bf16"),
        dict(name="block norm 16384 x 2048 bf16", op="block_norm", rows=16384, width=2048, x="bf16", o="bf16", gate="rows", y="bf16"),
    ]


def _size(rng, low, high):
    """Spread over the logarithm; one in three as it falls, the others rounded to a multiple of 16 where that leaves something."""
    n = int(round(low * (high / low) ** rng.random()))
    if rng.random() < 2 / 3 and n > 16:
        n = (n + 8) // 16 * 16
    return max(low, min(high, n))


def _seconds(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.4e15)


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend", "block_norm"])
    if op == "plan":
        return dict(op=op, nseq=_size(rng, 1, 2048), most=rng.choice([1, 1, 4, 64, 2048]), pages=rng.choice([64, 128, 200]))
    dim = rng.choice([32, 40, 48, 64, 64, 80, 96, 100, 128, 128, 128, 192, 256])
    if op == "append":
        while True:
            c = dict(op=op, rows=_size(rng, 1, 65536), kv_heads=rng.choice([1, 2, 4, 8, 16]), dk=dim, dv=rng.choice([dim, dim, 64, 128]), type=rng.choice(["f32", "bf16"]))
            if c["rows"] * c["kv_heads"] * (c["dk"] + c["dv"]) <= 65536 * 4 * 128:
                return c
    if op == "block_norm":
        while True:
            c = dict(op=op, rows=_size(rng, 1, 32768), width=_size(rng, 16, 16384), x=rng.choice(["f32", "bf16"]), o=rng.choice(["f32", "bf16"]),
                     gate=rng.choice(["none", "one", "rows"]), y=rng.choice(["f32", "bf16"]))
            if c["rows"] * c["width"] <= 16384 * 2048:
                return c
    top = max(_seconds(c) for c in listed())
    while True:
        kv_heads = rng.choice([1, 2, 4, 8, 16])
        new = rng.choice([1, 1, 1, 2, 5, _size(rng, 1, 2048)])
        c = dict(op=op, nseq=_size(rng, 1, 512), new=new, held=_size(rng, 1, 32000) - 1, even=rng.random() < 0.5, heads=kv_heads * rng.choice([1, 2, 4, 5, 8, 16]),
                 kv_heads=kv_heads, dk=dim, dv=rng.choice([dim, dim, 64, 128]), window=rng.choice([0, 0, 0, 128, 1000]), sink=rng.random() < 0.25, type=rng.choice(["f32", "bf16"]))
        length = c["held"] + new
        if _seconds(c) <= top and c["nseq"] * length * kv_heads * (c["dk"] + c["dv"]) <= 64 * 8192 * 8 * 256 and c["nseq"] * new * length * c["heads"] <= 1 << 29:
            return c


def _lengths(case):
    """Tokens that each sequence holds before the call, and new ones: the same for every seed, so that a case is one amount of work."""
    rng, n = random.Random(case["nseq"] * 7919 + case["held"]), case["nseq"]
    if case["even"]:
        return [case["held"]] * n, [case["new"]] * n
    held = [int((case["held"] + 1) ** (1 - 0.5 * rng.random())) - 1 if i else case["held"] for i in range(n)]
    return held, [case["new"] if i % 3 == 0 else rng.randint(0 if case["new"] > 1 else 1, case["new"]) for i in range(n)]


def _plan_lengths(case):
    """New tokens of each sequence: one for most, up to `most` for one in eight, none for some; -1 where the request has ended."""
    rng, most = random.Random(case["nseq"] * 104729 + case["most"]), case["most"]
    kinds = [rng.random() for _ in range(case["nseq"])]
    return [1 if most == 1 or k < 0.75 else -1 if k > 0.97 else 0 if k > 0.875 else max(1, int(most ** rng.random())) for k in kinds]


def _up(n, k):
    return (n + k - 1) // k * k


def _groups(d):
    return (d + 31) // 32


def _block(dk, dv):
    """Bytes of a page's block of one head."""
    return (_groups(dk) + _groups(dv)) * PAGE * 18


def _scale_up(m):
    """m / 7 rounded up to bf16 (m >= 2^-100), as fp32."""
    bits = (m / 7).view(torch.int32)
    return ((bits + 0xFFFF) & ~0xFFFF).view(torch.float32)


def _codes(t):
    """Numbers [..., d] to (codes 1 .. 15 of [..., groups, 32], 8 behind the last number, scales [..., groups] fp32)."""
    d = t.shape[-1]
    t = torch.nn.functional.pad(t.float(), (0, _groups(d) * 32 - d)).unflatten(-1, (-1, 32))
    s = _scale_up(t.abs().amax(-1).clamp(min=LEAST))
    return torch.round(t / s[..., None]).to(torch.uint8) + 8, s


KEY_ORDER = [0, 2, 4, 6, 1, 3, 5, 7]     # nibble i of a word of keys is number KEY_ORDER[i]
KEY_PLACE = [0, 4, 1, 5, 2, 6, 3, 7]     # number e of a word of keys is nibble KEY_PLACE[e]


def _pages_of(t, keys):
    """Numbers [pages, 64 tokens, heads, d] as the bytes of their part of the blocks: [pages, heads, bytes]."""
    n, s = _codes(t)
    if keys:
        n = n.unflatten(-1, (4, 8))[..., KEY_ORDER].flatten(-2)
    n = n[..., 0::2] | (n[..., 1::2] << 4)
    pages, _, heads = t.shape[:3]
    return torch.cat([n.permute(0, 2, 3, 1, 4).reshape(pages, heads, -1), s.bfloat16().permute(0, 2, 3, 1).contiguous().view(torch.uint8).reshape(pages, heads, -1)], dim=-1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    if case["op"] == "plan":
        nseq, width = case["nseq"], case["pages"]
        new = _plan_lengths(case)
        room = torch.tensor([width * PAGE - max(n, 0) for n in new], device="cuda")
        # half of the tables are filled at most, and one request in sixteen has just come
        held = (torch.rand(nseq, generator=gen, device="cuda") * torch.clamp(room, max=width * PAGE // 2)).int()
        held = torch.where(torch.rand(nseq, generator=gen, device="cuda") < 1 / 16, 0, held).int()
        s["len"], s["tokens"] = torch.tensor(new, device="cuda", dtype=torch.int32), held
        pages = (held + PAGE - 1) // PAGE
        first = torch.cumsum(pages, 0) - pages
        s["n_pages"] = nseq * width
        ids = torch.randperm(s["n_pages"], generator=gen, device="cuda").int()
        place = torch.arange(width, device="cuda")[None, :]
        s["table"] = torch.where(place < pages[:, None], ids[(first[:, None] + place).clamp(max=s["n_pages"] - 1)], -1).int().contiguous()
        used = int(pages.sum())
        s["free"] = torch.full((s["n_pages"],), -1, device="cuda", dtype=torch.int32)
        s["free"][:s["n_pages"] - used] = ids[used:]
        s["pool"] = torch.tensor([s["n_pages"] - used, 0], device="cuda", dtype=torch.int32)
        s["rows"] = _up(sum(max(n, 0) for n in new) + 1, 64)
        s["tokens_after"], s["pool_after"] = torch.zeros_like(held), torch.zeros_like(s["pool"])
        s["row_start"] = torch.zeros(nseq + 1, device="cuda", dtype=torch.int32)
        s["pos"], s["slot"] = torch.zeros(s["rows"], device="cuda", dtype=torch.int32), torch.zeros(s["rows"], device="cuda", dtype=torch.int32)
        return s
    if case["op"] == "block_norm":
        rows, width = case["rows"], case["width"]
        ld = _up(width, 8)
        # a few channels of a residual stream are much larger than the others
        factor = torch.where(torch.rand(width, generator=gen, device="cuda") < 0.01, 8.0, 1.0)

        def numbers(n, kind, by=1.0):
            buf = torch.zeros(n, ld, device="cuda", dtype=TYPES[kind])
            buf[:, :width] = normal(n, width) * by
            return buf[:, :width]

        s["xs"], s["os"] = numbers(rows, case["x"], factor), numbers(rows, case["o"])
        s["gates"] = None if case["gate"] == "none" else numbers(1 if case["gate"] == "one" else rows, case["o"])
        s["post"], s["pre"] = 1 + 0.1 * normal(width), 1 + 0.1 * normal(width)
        s["ys"] = numbers(rows, case["y"], 0.0)
        return s
    heads, dk, dv, dtype = case["kv_heads"], case["dk"], case["dv"], TYPES[case["type"]]
    if case["op"] == "append":
        rows = case["rows"]
        ldk, ldv = _up(heads * dk, 8), _up(heads * dv, 8)
        # a few channels of the keys are much larger than the others
        factor = torch.where(torch.rand(ldk, generator=gen, device="cuda") < 0.02, 6.0, 1.0)
        s["k"], s["v"] = (normal(rows, ldk) * factor).to(dtype), normal(rows, ldv, dtype=dtype)
        s["n_pages"] = (rows + PAGE - 1) // PAGE + 8
        # sequences' runs of tokens: whole pages in any order, the slots of a page in their order
        order = torch.randperm(s["n_pages"], generator=gen, device="cuda")
        at = torch.arange(rows, device="cuda")
        s["slot"] = (order[at // PAGE] * PAGE + at % PAGE).int()
        s["kv"] = torch.zeros(s["n_pages"], heads, _block(dk, dv), device="cuda", dtype=torch.uint8)
        s["k_out"], s["v_out"] = torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
        return s
    held, new = _lengths(case)
    nseq, total = case["nseq"], [a + b for a, b in zip(held, new)]
    s["longest"], s["max_new"], s["rows"] = max(total), max(new), sum(new)
    need = [(t + PAGE - 1) // PAGE for t in total]
    s["pages_per_seq"], s["n_pages"] = max(need) + 1, sum(need) + 4
    pages = torch.tensor(need, device="cuda")
    order = torch.randperm(s["n_pages"], generator=gen, device="cuda").int()
    place = torch.arange(s["pages_per_seq"], device="cuda")[None, :]
    spot = (torch.cumsum(pages, 0) - pages)[:, None] + place
    s["table"] = torch.where(place < pages[:, None], order[spot.clamp(max=s["n_pages"] - 1)], -1).int().contiguous()
    starts = torch.tensor([0] + new, device="cuda")
    s["row_start"] = torch.cumsum(starts, 0).int()
    s["tokens"] = torch.tensor(total, device="cuda", dtype=torch.int32)
    s["kv"] = torch.empty(s["n_pages"], heads, _block(dk, dv), device="cuda", dtype=torch.uint8)
    part = max(1, (1 << 26) // (PAGE * heads * (dk + dv)))
    split = _groups(dk) * PAGE * 18
    for a in range(0, s["n_pages"], part):
        n = min(part, s["n_pages"] - a)
        s["kv"][a:a + n, :, :split] = _pages_of(normal(n, PAGE, heads, dk), True)
        s["kv"][a:a + n, :, split:] = _pages_of(normal(n, PAGE, heads, dv), False)
    # queries whose scores spread as those of trained models do: a few keys take most of the weight
    s["q"] = (normal(s["rows"], case["heads"] * dk) * 1.5).to(dtype)
    s["y"] = torch.zeros(s["rows"], case["heads"] * dv, device="cuda", dtype=dtype)
    # what the library keeps of a call's parts until they are joined: this many bytes at most, zero before the first call
    s["work"] = torch.zeros(64 << 20, device="cuda", dtype=torch.uint8)
    return s


# ---- plain forms

def _plain_plan(s):
    width, rows = s["table"].shape[1], s["rows"]
    new, gone, held = s["len"].clamp(min=0), s["len"] < 0, s["tokens"]
    after = torch.where(gone, 0, held + new)
    before_pages, after_pages = (held + PAGE - 1) // PAGE, (after + PAGE - 1) // PAGE
    taken = torch.where(gone, 0, after_pages - before_pages)
    given = torch.where(gone, before_pages, 0)
    zero = torch.zeros(1, device="cuda", dtype=torch.int64)
    row_start = torch.cat([zero, torch.cumsum(new, 0)])
    take_start, give_start = torch.cumsum(taken, 0) - taken, torch.cumsum(given, 0) - given
    n_free, n_given, n_taken = s["pool"][0], given.sum(), taken.sum()
    # the free pages, and behind them those that come back, in the order of their sequences
    place = torch.arange(width, device="cuda")[None, :]
    stack = torch.cat([s["free"], zero.int()])
    to = torch.where(place < given[:, None], n_free + give_start[:, None] + place, s["n_pages"])
    stack = stack.scatter(0, to.flatten().long(), s["table"].flatten())[:-1]
    fresh = (place >= before_pages[:, None]) & (place < after_pages[:, None]) & ~gone[:, None]
    of = n_free + n_given - 1 - (take_start[:, None] + place - before_pages[:, None])
    table = torch.where(fresh, stack[of.clamp(min=0, max=s["n_pages"] - 1)], s["table"])
    left = n_free + n_given - n_taken
    at = torch.arange(s["n_pages"], device="cuda")
    free = torch.where((at >= n_free) & (at < left), stack, s["free"])
    row = torch.arange(rows, device="cuda")
    seq = (torch.searchsorted(row_start, row, right=True) - 1).clamp(max=s["nseq"] - 1)
    lives = row < row_start[-1]
    pos = held[seq] + row - row_start[seq]
    slot = table[seq, (pos // PAGE).clamp(max=width - 1)] * PAGE + pos % PAGE
    return {"row_start": row_start.int(), "pos": torch.where(lives, pos, -1).int(), "slot": torch.where(lives, slot, -1).int(), "table": table, "tokens": after.int(),
            "free": free, "pool": torch.stack([left, s["pool"][1]]).int()}


def _values(kv, groups, d, keys):
    """The numbers that [..., 64 tokens] of one part of the blocks stand for: bytes [..., heads, groups * 64 * 18] to [..., heads, 64, d] fp32."""
    n = kv[..., :groups * PAGE * 16].unflatten(-1, (groups, PAGE, 16))
    n = torch.stack([n & 15, n >> 4], dim=-1).flatten(-2)
    if keys:
        n = n.unflatten(-1, (4, 8))[..., KEY_PLACE].flatten(-2)
    s = kv[..., groups * PAGE * 16:].contiguous().view(torch.bfloat16).unflatten(-1, (groups, PAGE))
    t = (n.float() - 8) * s.float()[..., None]
    return t.transpose(-3, -2).flatten(-2)[..., :d]


def _held(t, heads, d):
    """Rows t as the cache holds them."""
    n, scale = _codes(t[:, :heads * d].unflatten(-1, (heads, d)))
    return ((n.float() - 8) * scale[..., None]).flatten(-2)[..., :d].flatten(-2).to(t.dtype)


def _plain_append(s):
    return {"k": _held(s["k"], s["kv_heads"], s["dk"]), "v": _held(s["v"], s["kv_heads"], s["dv"])}


def _plain_attend(s):
    nseq, heads, kv_heads, dk, dv, n = s["nseq"], s["heads"], s["kv_heads"], s["dk"], s["dv"], s["max_new"]
    split = _groups(dk) * PAGE * 18
    pages = s["kv"][s["table"][:, :(s["longest"] + PAGE - 1) // PAGE].clamp(min=0)]          # [nseq, pages, kv_heads, bytes]
    k = _values(pages[..., :split], _groups(dk), dk, True).transpose(1, 2).flatten(2, 3)     # [nseq, kv_heads, tokens, dk]
    v = _values(pages[..., split:], _groups(dv), dv, False).transpose(1, 2).flatten(2, 3)
    start, new = s["row_start"][:-1].long(), (s["row_start"][1:] - s["row_start"][:-1]).long()
    i = torch.arange(n, device="cuda")
    row = torch.where(i < new[:, None], start[:, None] + i, s["rows"] - 1)                   # [nseq, n]
    q = s["q"].float()[row].unflatten(-1, (kv_heads, heads // kv_heads, dk)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    x = torch.matmul(q, k.transpose(-1, -2)).unflatten(2, (heads // kv_heads, n)) * dk ** -0.5
    pos = (s["tokens"].long() - new)[:, None] + i
    at = torch.arange(x.shape[-1], device="cuda")
    seen = at <= pos[..., None]
    if s["window"]:
        seen = seen & (at > pos[..., None] - s["window"])
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    if s["sink"]:
        m = m.clamp(min=0)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    if s["sink"]:
        total = total + torch.exp(-m)
    y = torch.matmul((p / total).flatten(2, 3), v).unflatten(2, (heads // kv_heads, n)).permute(0, 3, 1, 2, 4).flatten(2)
    return y[i < new[:, None]].to(s["q"].dtype)


def _plain_block_norm(s):
    o = s["os"].float()
    o = o / torch.sqrt((o * o).mean(-1, keepdim=True) + EPS) * s["post"]
    if s["gates"] is not None:
        o = o * s["gates"].float()
    s["xs"].copy_(s["xs"].float() + 0.5 * o)
    t = s["xs"].float()
    return {"x": s["xs"], "y": (t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * s["pre"]).to(s["ys"].dtype)}


# ---- the library's calls

def _dtype(t):
    return 1 if t.dtype == torch.bfloat16 else 0


def _library(s):
    import lumi_b200
    lib, check = lumi_b200.lib(), lumi_b200.api.check
    stream = torch.cuda.current_stream().cuda_stream
    if s["op"] == "plan":
        check(lib.lumi_k_page_plan(s["tokens"].data_ptr(), s["len"].data_ptr(), s["nseq"], s["table"].data_ptr(), s["table"].shape[1], s["free"].data_ptr(), s["n_pages"],
                                   s["pool"].data_ptr(), s["pool_after"].data_ptr(), s["tokens_after"].data_ptr(), s["row_start"].data_ptr(), s["pos"].data_ptr(),
                                   s["slot"].data_ptr(), s["rows"], stream))
        return {"row_start": s["row_start"], "pos": s["pos"], "slot": s["slot"], "table": s["table"], "tokens": s["tokens_after"], "free": s["free"], "pool": s["pool_after"]}
    if s["op"] == "block_norm":
        x, o, g, y = s["xs"], s["os"], s["gates"], s["ys"]
        check(lib.lumi_k_block_norm(x.data_ptr(), _dtype(x), x.stride(0), o.data_ptr(), _dtype(o), o.stride(0), s["post"].data_ptr(), 0 if g is None else g.data_ptr(),
                                    0 if g is None or g.shape[0] == 1 and s["gate"] == "one" else g.stride(0), 0.5, s["pre"].data_ptr(), y.data_ptr(), _dtype(y), y.stride(0),
                                    s["rows"], s["width"], EPS, stream))
        return {"x": x, "y": y}
    heads, dk, dv = s["kv_heads"], s["dk"], s["dv"]
    if s["op"] == "append":
        k, v, k2, v2, at, rows = s["k"], s["v"], s["k_out"], s["v_out"], s["slot"].data_ptr(), s["rows"]
        check(lib.lumi_k_kv4_append(k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), _dtype(k), at, s["kv"].data_ptr(), s["n_pages"], heads, dk, dv, rows, stream))
        check(lib.lumi_k_kv4_read(s["kv"].data_ptr(), s["n_pages"], at, k2.data_ptr(), k2.stride(0), v2.data_ptr(), v2.stride(0), _dtype(k2), heads, dk, dv, rows, stream))
        return {"k": k2[:, :heads * dk], "v": v2[:, :heads * dv]}
    q, y = s["q"], s["y"]
    check(lib.lumi_k_kv4_attention(q.data_ptr(), q.stride(0), _dtype(q), s["kv"].data_ptr(), s["n_pages"], s["table"].data_ptr(), s["pages_per_seq"], s["row_start"].data_ptr(),
                                   s["tokens"].data_ptr(), y.data_ptr(), y.stride(0), s["heads"], heads, dk, dv, s["window"], dk ** -0.5, int(s["sink"]), s["nseq"], s["rows"],
                                   s["max_new"], s["work"].data_ptr(), s["work"].numel(), 0, stream))
    return y


def run(state):
    if own:
        return _library(state)
    return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend, "block_norm": _plain_block_norm}[state["op"]](state)


# ---- the definitions in 64 bits

def _exact_plan(s):
    """Sequence after sequence on the host."""
    table, free, tokens = s["table"].cpu().numpy().copy(), s["free"].cpu().numpy().copy(), s["tokens"].cpu().tolist()
    n_free = int(s["pool"][0])
    stack, rows, starts = free[:n_free].tolist(), [], [0]
    new = s["len"].cpu().tolist()
    for i, n in enumerate(new):
        if n < 0:
            stack += table[i, :(tokens[i] + PAGE - 1) // PAGE].tolist()
            tokens[i] = 0
    for i, n in enumerate(new):
        for _ in range(max(n, 0)):
            if tokens[i] % PAGE == 0:
                table[i, tokens[i] // PAGE] = stack.pop()
            rows.append((tokens[i], int(table[i, tokens[i] // PAGE]) * PAGE + tokens[i] % PAGE))
            tokens[i] += 1
        starts.append(len(rows))
    if len(stack) > n_free:
        free[n_free:len(stack)] = stack[n_free:]
    rows += [(-1, -1)] * (s["rows"] - len(rows))
    dev = lambda a: torch.tensor(a, device="cuda", dtype=torch.int32)
    return {"row_start": dev(starts), "pos": dev([r[0] for r in rows]), "slot": dev([r[1] for r in rows]), "table": dev(table), "tokens": dev(tokens), "free": dev(free),
            "pool": dev([len(stack), 0])}


def _exact_held(t, heads, d):
    """What the cache holds of rows t: group after group."""
    t = t[:, :heads * d].reshape(-1, heads, d)
    out = torch.empty(t.shape, device="cuda", dtype=torch.float64)
    for a in range(0, d, 32):
        part = t[..., a:a + 32].to(torch.float32)
        largest = part.abs().max(-1, keepdim=True).values
        seventh = torch.maximum(largest, torch.full_like(largest, LEAST)) / 7
        step = seventh.to(torch.bfloat16)
        low = step.float() < seventh                                        # the next bf16 above
        step = torch.where(low, (step.view(torch.int16) + 1).view(torch.bfloat16), step).float()
        out[..., a:a + 32] = torch.round(part / step).double() * step.double()
    return out.reshape(t.shape[0], heads * d)


def _exact_numbers(blocks, first, d, keys):
    """[pages, heads, bytes] to [heads, pages * 64, d]: every number looked up by its own byte."""
    dim, tok = torch.arange(d, device="cuda"), torch.arange(PAGE, device="cuda")
    e = dim % 8
    nibble = dim % 32 // 8 * 8 + e // 2 + e % 2 * 4 if keys else dim % 32
    byte = first + dim // 32 * (PAGE * 16) + nibble // 2 + tok[:, None] * 16
    code = (blocks[:, :, byte].to(torch.int32) >> (nibble % 2 * 4)) & 15
    at = first + _groups(d) * PAGE * 16 + dim // 32 * (PAGE * 2) + tok[:, None] * 2
    bits = blocks[:, :, at].to(torch.int32) << 16 | blocks[:, :, at + 1].to(torch.int32) << 24
    t = (code - 8).double() * bits.view(torch.float32).double()
    return t.transpose(0, 1).reshape(blocks.shape[1], -1, d)


def _exact_attend(s):
    held, new = _lengths(s)
    group, out = s["heads"] // s["kv_heads"], []
    for b in range(s["nseq"]):
        total, first = held[b] + new[b], sum(new[:b])
        if new[b] == 0:
            continue
        blocks = s["kv"][s["table"][b, :(total + PAGE - 1) // PAGE].long()]
        k = _exact_numbers(blocks, 0, s["dk"], True)[:, :total]
        v = _exact_numbers(blocks, _groups(s["dk"]) * PAGE * 18, s["dv"], False)[:, :total]
        q = s["q"][first:first + new[b]].double().reshape(new[b], s["kv_heads"], group, s["dk"]).permute(1, 2, 0, 3)
        ages = torch.arange(held[b], total, device="cuda")[:, None] - torch.arange(total, device="cuda")[None, :]
        hidden = (ages < 0) | (ages >= s["window"] if s["window"] else ages < 0)
        y = torch.empty(s["kv_heads"], group, new[b], s["dv"], device="cuda", dtype=torch.float64)
        for h in range(s["kv_heads"]):
            x = torch.einsum("gnd,ld->gnl", q[h], k[h]) / math.sqrt(s["dk"])
            x = x.masked_fill(hidden, -math.inf)
            if s["sink"]:
                x = torch.cat([x, torch.zeros_like(x[..., :1])], -1)
            y[h] = torch.softmax(x, -1)[..., :total] @ v[h]
        out.append(y.permute(2, 0, 1, 3).reshape(new[b], -1))
    return torch.cat(out)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return _exact_plan(s)
    if case["op"] == "append":
        return {"k": _exact_held(s["k"], s["kv_heads"], s["dk"]), "v": _exact_held(s["v"], s["kv_heads"], s["dv"])}
    if case["op"] == "attend":
        return _exact_attend(s)
    o = s["os"].double()
    add = o * (o.pow(2).sum(1, keepdim=True) / case["width"] + EPS).rsqrt() * s["post"].double() / 2
    x = s["xs"].double() + (add if s["gates"] is None else add * s["gates"].double())
    seen = x.to(torch.float32).to(torch.bfloat16).double() if case["x"] == "bf16" else x     # the stored stream is what the second norm sees
    return {"x": x, "y": seen * (seen.pow(2).sum(1, keepdim=True) / case["width"] + EPS).rsqrt() * s["pre"].double()}


def work(case):
    """Every input read once, every output written once; of the cache, the tokens that some row of the call sees."""
    if case["op"] == "plan":
        new = sum(max(n, 0) for n in _plan_lengths(case))
        # lengths in and out, starts, a position and a slot per row, the table's entry that a slot is of, new entries and the free pages they come from
        return {"bytes": 16 * case["nseq"] + 8 * new + 12 * max(1, new // PAGE), "flops": 4 * new}
    if case["op"] == "block_norm":
        n, e = case["rows"] * case["width"], {k: TYPES[case[k]].itemsize for k in ("x", "o", "y")}
        gate = {"none": 0, "one": case["width"], "rows": n}[case["gate"]] * e["o"]
        return {"bytes": n * (2 * e["x"] + e["o"] + e["y"]) + gate + 8 * case["width"], "flops": 10 * n}
    heads, dk, dv, e = case["kv_heads"], case["dk"], case["dv"], TYPES[case["type"]].itemsize
    token = heads * (math.ceil(dk / 2) + math.ceil(dv / 2) + 2 * (_groups(dk) + _groups(dv)))
    if case["op"] == "append":
        # rows in, codes and scales out, and both the other way round
        return {"bytes": case["rows"] * 2 * (heads * (dk + dv) * e + token + 4), "flops": 8 * case["rows"] * heads * (dk + dv)}
    held, new = _lengths(case)
    tokens = pairs = 0
    for h, n in zip(held, new):
        if n == 0:
            continue
        w = case["window"] or h + n
        tokens += min(h + n, w + n - 1)
        # row i sees min(h + i + 1, w) tokens
        short = max(0, min(n, w - h))
        pairs += short * h + short * (short + 1) // 2 + (n - short) * w
    return {"bytes": tokens * token + sum(new) * case["heads"] * (dk + dv) * e, "flops": 2 * pairs * case["heads"] * (dk + dv)}
