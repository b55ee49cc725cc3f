"""The cache in 4 bits in 64-bit numpy: its layout byte by byte, plans of pages, and attention over what the bytes stand for.  Shared by the tests of the calls."""
import numpy as np

PAGE, GROUP = 64, 32


def groups(d):
    return (d + GROUP - 1) // GROUP


def block_bytes(dk, dv):
    return (groups(dk) + groups(dv)) * PAGE * 18


def bf16_up(x):
    """Positive fp32 numbers rounded up to bf16."""
    bits = np.asarray(x, np.float32).view(np.uint32)
    return ((bits + np.uint32(0xFFFF)) & np.uint32(0xFFFF0000)).view(np.float32)


def quantise(t):
    """[..., d] fp32 to (codes [..., d] int, scales [..., groups] fp32)."""
    t = np.asarray(t, np.float32)
    codes = np.full(t.shape, 8, np.int64)
    scales = np.empty(t.shape[:-1] + (groups(t.shape[-1]),), np.float32)
    for g in range(scales.shape[-1]):
        part = t[..., g * GROUP:(g + 1) * GROUP]
        good = np.isfinite(part).all(-1)
        m = np.maximum(np.where(good, np.abs(part).max(-1), 1), np.float32(2.0 ** -100)).astype(np.float32)
        s = bf16_up(m * (np.float32(1) / np.float32(7)))
        with np.errstate(invalid="ignore"):
            n = 8 + np.rint((part / s[..., None]).astype(np.float32))
        codes[..., g * GROUP:(g + 1) * GROUP] = np.where(good[..., None], n, 8)
        scales[..., g] = np.where(good, s, np.nan)
    return codes, scales


def values(codes, scales):
    return (codes - 8).astype(np.float64) * np.repeat(scales.astype(np.float64), GROUP, -1)[..., :codes.shape[-1]]


def nibble(d, keys):
    i = d % GROUP
    return i // 8 * 8 + i % 8 // 2 + 4 * (i % 2) if keys else i


def write(cache, slot, head, k, v):
    """One token and head into cache [pages, heads, block] uint8 (of a fresh or an older token)."""
    at = 0
    for t, keys in ((k, True), (v, False)):
        codes, scales = quantise(t)
        page, tok, g_all = slot // PAGE, slot % PAGE, groups(len(t))
        for d in range(g_all * GROUP):
            n = int(codes[d]) if d < len(t) else 8
            b = at + d // GROUP * PAGE * 16 + tok * 16 + nibble(d, keys) // 2
            sh = 4 * (nibble(d, keys) % 2)
            cache[page, head, b] = cache[page, head, b] & (0xF0 >> sh) | n << sh
        for g in range(g_all):
            b = at + g_all * PAGE * 16 + g * PAGE * 2 + tok * 2
            bits = int(np.float32(scales[g]).view(np.uint32)) >> 16 if np.isfinite(scales[g]) else 0x7FC0
            cache[page, head, b:b + 2] = (bits & 255, bits >> 8)
        at += g_all * PAGE * 18


def read(cache, slots, dk, dv):
    """(keys [slots, heads, dk], values [slots, heads, dv]) in 64 bits."""
    slots = np.asarray(slots)
    blocks = cache[slots // PAGE]                                  # [slots, heads, block]
    tok = slots % PAGE
    out, at = [], 0
    for d, keys in ((dk, True), (dv, False)):
        dim, g = np.arange(d), groups(d)
        nib = np.array([nibble(i, keys) for i in dim])
        b = at + dim // GROUP * PAGE * 16 + nib // 2 + tok[:, None] * 16
        n = np.take_along_axis(blocks, np.broadcast_to(b[:, None], blocks.shape[:2] + (d,)), 2) >> (4 * (nib % 2)) & 15
        sb = at + g * PAGE * 16 + dim // GROUP * PAGE * 2 + tok[:, None] * 2
        lo = np.take_along_axis(blocks, np.broadcast_to(sb[:, None], blocks.shape[:2] + (d,)), 2).astype(np.uint32)
        hi = np.take_along_axis(blocks, np.broadcast_to(sb[:, None] + 1, blocks.shape[:2] + (d,)), 2).astype(np.uint32)
        out.append((n.astype(np.float64) - 8) * (lo << 16 | hi << 24).astype(np.uint32).view(np.float32).astype(np.float64))
        at += g * PAGE * 18
    return out


def plan(tokens, new, table, free, pool, n_pages, rows):
    """lumi_k_page_plan on lists, sequence after sequence: (tokens, table, free, pool, row_start, pos, slot)."""
    width, bad = table.shape[1], 0
    for h, n in zip(tokens, new):
        if h < 0 or h + max(n, 0) > width * PAGE:
            bad |= 2
    if not bad:
        given = sum((h + PAGE - 1) // PAGE for h, n in zip(tokens, new) if n < 0)
        taken = sum((h + n + PAGE - 1) // PAGE - (h + PAGE - 1) // PAGE for h, n in zip(tokens, new) if n >= 0)
        if not 0 <= pool[0] <= n_pages or taken > pool[0] + given or pool[0] + given - taken > n_pages:
            bad |= 1
        if sum(max(n, 0) for n in new) > rows:
            bad |= 4
    if bad:
        return list(tokens), table.copy(), free.copy(), [pool[0], pool[1] | bad], [0] * (len(tokens) + 1), [-1] * rows, [-1] * rows
    tokens, table, out = list(tokens), table.copy(), free.copy()
    stack = [int(p) for p in free[:pool[0]]]
    for s, n in enumerate(new):
        if n < 0:
            stack += [int(p) for p in table[s, :(tokens[s] + PAGE - 1) // PAGE]]
            tokens[s] = 0
    pos, slot, start = [], [], [0]
    for s, n in enumerate(new):
        for _ in range(max(n, 0)):
            i = tokens[s] // PAGE
            if tokens[s] % PAGE == 0:
                table[s, i] = stack.pop()
            pos.append(tokens[s])
            slot.append(int(table[s, i]) * PAGE + tokens[s] % PAGE)
            tokens[s] += 1
        start.append(len(pos))
    out[pool[0]:len(stack)] = stack[pool[0]:]
    return tokens, table, out, [len(stack), pool[1]], start, pos + [-1] * (rows - len(pos)), slot + [-1] * (rows - len(slot))


def attend(q, k, v, first, scale, window, sink):
    """Rows q [n, heads, dk] at positions first .. first + n - 1 over keys k [tokens, kv_heads, dk] and values [tokens, kv_heads, dv]; tokens that are not there have NaN keys in
    `hidden` rows of neither.  Returns (y [n, heads, dv], the largest scale * sum |q k| a row meets [n, heads])."""
    n, heads, _ = q.shape
    group = heads // k.shape[1]
    y, spread = np.zeros((n, heads, v.shape[2])), np.zeros((n, heads))
    for i in range(n):
        pos = first + i
        lo = max(0, pos - window + 1) if window else 0
        for h in range(heads):
            kk, vv = k[lo:pos + 1, h // group], v[lo:pos + 1, h // group]
            x = kk @ q[i, h] * scale
            m = max([0.0] if sink else [-np.inf], default=-np.inf)
            m = max(m, x.max(initial=-np.inf))
            p = np.exp(x - m)
            total = p.sum() + (np.exp(-m) if sink else 0.0)
            y[i, h] = p @ vv / total if total else 0.0
            spread[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max(initial=0.0) * abs(scale)
    return y, spread
