"""Page plans, and rows into the cache in 4 bits and back, against the byte-by-byte reference."""
import numpy as np
import pytest
import torch

import kv4_reference as ref
import lumi_b200

pytestmark = pytest.mark.gpu
PAGE = 64


def stream():
    return torch.cuda.current_stream().cuda_stream


def ok(status):
    lumi_b200.api.check(status)


def dev(a, dtype=torch.int32):
    return torch.tensor(np.asarray(a), device="cuda", dtype=dtype)


class Plan:
    """The arrays of one plan; guard values behind every output."""

    def __init__(self, tokens, new, width, n_pages, rows, rng, spare=0):
        self.tokens, self.new, self.width, self.n_pages, self.rows = [int(t) for t in tokens], [int(n) for n in new], width, n_pages, rows
        ids = rng.permutation(n_pages)
        self.table = np.full((len(tokens), width), -7, np.int64)
        used = 0
        for s, t in enumerate(tokens):
            need = max(0, min(width, (t + PAGE - 1) // PAGE))
            self.table[s, :need] = ids[used:used + need]
            used += need
        self.free = np.full(n_pages, -9, np.int64)
        self.free[:n_pages - used - spare] = ids[used:n_pages - spare]
        self.pool = [n_pages - used - spare, 0]

    def run(self, in_place=False, launch=None):
        d = dict(tokens=dev(self.tokens + [77]), new=dev(self.new + [5]), table=dev(np.concatenate([self.table.ravel(), [-3]])), free=dev(np.append(self.free, -3)), pool=dev(self.pool + [-3]),
                 row_start=dev([-3] * (len(self.tokens) + 2)), pos=dev([-3] * (self.rows + 1)), slot=dev([-3] * (self.rows + 1)))
        d["tokens_after"] = d["tokens"] if in_place else dev([-3] * (len(self.tokens) + 1))
        d["pool_after"] = d["pool"] if in_place else dev([-3] * 3)
        self.d = d
        (launch or self.launch)()
        torch.cuda.synchronize()
        return self.results()

    def launch(self):
        d = self.d
        ok(lumi_b200.lib().lumi_k_page_plan(d["tokens"].data_ptr(), d["new"].data_ptr(), len(self.tokens), d["table"].data_ptr(), self.width, d["free"].data_ptr(), self.n_pages,
                                            d["pool"].data_ptr(), d["pool_after"].data_ptr(), d["tokens_after"].data_ptr(), d["row_start"].data_ptr(), d["pos"].data_ptr(),
                                            d["slot"].data_ptr(), self.rows, stream()))

    def results(self):
        d = {k: v.cpu().numpy() for k, v in self.d.items()}
        assert d["row_start"][-1] == -3 and d["pos"][-1] == -3 and d["slot"][-1] == -3 and d["table"][-1] == -3 and d["free"][-1] == -3 and d["pool_after"][2] == -3
        assert d["tokens_after"][-1] in (77, -3) and d["new"][-1] == 5
        return [d["tokens_after"][:-1], d["table"][:-1].reshape(self.table.shape), d["free"][:-1], d["pool_after"][:2], d["row_start"][:-1], d["pos"][:-1], d["slot"][:-1]]

    def expected(self):
        return ref.plan(self.tokens, self.new, self.table, self.free, self.pool, self.n_pages, self.rows)

    def check(self, **k):
        for got, want, what in zip(self.run(**k), self.expected(), ("tokens", "table", "free", "pool", "row_start", "pos", "slot")):
            assert np.array_equal(got, np.asarray(want).reshape(got.shape)), what


def lengths(nseq, most, width, rng):
    tokens = rng.integers(0, width * PAGE // 2, nseq)
    tokens[rng.random(nseq) < 0.2] = 0
    edge = rng.random(nseq) < 0.3
    tokens[edge] = tokens[edge] // PAGE * PAGE + rng.integers(0, 2, edge.sum()) * (PAGE - 1)
    kind = rng.random(nseq)
    new = np.where(kind < 0.5, 1, np.where(kind < 0.6, 0, np.where(kind < 0.75, -1 - rng.integers(0, 3, nseq), rng.integers(0, most + 1, nseq))))
    return tokens, new


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("nseq,most,width", [(1, 1, 1), (1, 200, 9), (3, 64, 5), (31, 130, 6), (200, 1, 4), (1024, 3, 4), (1500, 40, 8), (5000, 4, 4), (8192, 2, 3)])
def test_plans(nseq, most, width, in_place):
    rng = np.random.default_rng(nseq + most)
    tokens, new = lengths(nseq, min(most, width * PAGE // 2), width, rng)
    rows = int(np.maximum(new, 0).sum()) + (nseq * 7) % 50
    Plan(tokens, new, width, nseq * width + 5, rows, rng).check(in_place=in_place)


def test_no_sequences_and_no_rows():
    rng = np.random.default_rng(0)
    Plan([], [], 3, 4, 5, rng).check()
    Plan([10, 64], [0, -1], 3, 8, 0, rng).check()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("tokens,new,width,n_pages,rows,spare,bits", [
    ([64, 64, 1], [1, 1, 1], 4, 5, 8, 1, 1),         # one page free, two are needed
    ([64, 3], [65, 0], 2, 8, 200, 0, 2),             # 129 tokens in two pages
    ([64, -1], [1, 1], 2, 8, 8, 0, 2),               # no count of tokens
    ([64, 3], [4, 4], 3, 8, 7, 0, 4),                # eight rows, room for seven
    ([2 ** 31 - 1, 3], [2 ** 31 - 1, 4], 3, 8, 9, 0, 2)])
def test_plans_that_cannot_be(tokens, new, width, n_pages, rows, spare, bits, in_place):
    p = Plan([min(t, width * PAGE) for t in tokens], new, width, n_pages, rows, np.random.default_rng(1), spare)
    p.tokens = tokens
    assert p.expected()[3][1] == bits
    p.check(in_place=in_place)


def test_a_count_of_free_pages_that_is_none():
    for count in (-1, 9):
        p = Plan([1], [1], 2, 8, 4, np.random.default_rng(1))
        p.pool = [count, 16]
        got = p.run()
        assert list(got[3]) == [count, 17] and list(got[4]) == [0, 0] and list(got[0]) == [1]


def test_more_come_back_than_are_taken_and_the_other_way_round():
    rng = np.random.default_rng(2)
    Plan([300, 10, 64, 640, 0], [-1, 60, 1, -5, 100], 16, 80, 300, rng).check()
    Plan([100, 10, 64, 640, 0], [-1, 700, 1, 300, 500], 16, 80, 2000, rng, spare=20).check(in_place=True)


def test_a_captured_plan_goes_on_from_replay_to_replay():
    """In place: every replay adds its tokens, until a page is missing; then nothing changes but the bit."""
    rng = np.random.default_rng(3)
    p = Plan([60, 0, 190], [2, 1, 1], 8, 6, 16, rng)
    p.run(in_place=True, launch=lambda: None)
    d, table, pool, free, tokens = p.d, p.table.copy(), list(p.pool), p.free.copy(), list(p.tokens)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            p.launch()
        for _ in range(80):
            graph.replay()
            side.synchronize()
            tokens, table, free, pool, start, pos, slot = ref.plan(tokens, p.new, table, free, pool, p.n_pages, p.rows)
            got = p.results()
            for g, w in zip(got, (tokens, table, free, pool, start, pos, slot)):
                assert np.array_equal(g, np.asarray(w).reshape(g.shape))
    assert pool[1] == 1


# ---- rows into the cache and back
def numbers(shape, rng, kind="normal"):
    t = rng.standard_normal(shape).astype(np.float32)
    if kind == "wide":
        t *= np.exp2(rng.integers(-120, 120, shape[:1] + (1,) * (len(shape) - 1))).astype(np.float32)
    if kind == "zeros":
        t[::2] = 0
        t[1::4] *= np.float32(2.0 ** -110)
    if kind == "ties":
        t = np.rint(t * 6).astype(np.float32) / 2
        t[..., 0] = 7
    if kind == "none":
        t[0, ..., 3] = np.inf
        t[1, ..., 0] = np.nan
        t[2, ..., -1] = -np.inf
    return t


def rows_of(t, ld, dtype):
    """t [rows, heads, d] as rows of ld elements with NaN behind them: (buffer, row view)."""
    n, w = t.shape[0], t.shape[1] * t.shape[2]
    buf = torch.full((n, ld), float("nan"), device="cuda", dtype=dtype)
    buf[:, :w] = torch.tensor(t.reshape(n, w), device="cuda").to(dtype)
    return buf


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,heads,dk,dv,pad,kind", [
    (1, 1, 1, 1, 0, "normal"), (7, 2, 64, 64, 0, "normal"), (33, 4, 128, 128, 8, "normal"), (64, 3, 80, 100, 0, "normal"), (9, 2, 33, 40, 3, "normal"), (130, 1, 256, 32, 0, "normal"),
    (16, 5, 96, 192, 0, "wide"), (20, 2, 64, 48, 4, "zeros"), (40, 2, 64, 64, 0, "ties"), (12, 3, 40, 33, 1, "none")])
def test_rows_in_and_out(rows, heads, dk, dv, pad, kind, dtype):
    rng = np.random.default_rng(rows + dk)
    n_pages = rows // 8 + 2
    # slots anywhere, some rows without one
    slots = rng.permutation(n_pages * PAGE)[:rows]
    slots[rng.random(rows) < 0.1] = -1
    if rows > 8:
        slots[[1, 4]] = [n_pages * PAGE, 2 ** 31 - 1]
    kb, vb = rows_of(numbers((rows, heads, dk), rng, kind), heads * dk + pad, dtype), rows_of(numbers((rows, heads, dv), rng, kind), heads * dv + pad, dtype)
    cache = rng.integers(0, 256, (n_pages, heads, ref.block_bytes(dk, dv)), dtype=np.uint8)
    kv = torch.tensor(cache, device="cuda")
    at = dev(slots)
    lib, code = lumi_b200.lib(), int(dtype == torch.bfloat16)
    ok(lib.lumi_k_kv4_append(kb.data_ptr(), kb.stride(0), vb.data_ptr(), vb.stride(0), code, at.data_ptr(), kv.data_ptr(), n_pages, heads, dk, dv, rows, stream()))
    torch.cuda.synchronize()
    k, v = kb.float().cpu().numpy()[:, :heads * dk].reshape(rows, heads, dk), vb.float().cpu().numpy()[:, :heads * dv].reshape(rows, heads, dv)
    live = [(i, s) for i, s in enumerate(slots) if 0 <= s < n_pages * PAGE]
    for i, s in live:
        for h in range(heads):
            ref.write(cache, s, h, k[i, h], v[i, h])
    assert np.array_equal(kv.cpu().numpy(), cache)                    # every byte, those of other slots among them
    for out_dtype in (torch.float32, torch.bfloat16):
        ko, vo = torch.full((rows, heads * dk + pad), -5.0, device="cuda", dtype=out_dtype), torch.full((rows, heads * dv + pad), -5.0, device="cuda", dtype=out_dtype)
        ok(lib.lumi_k_kv4_read(kv.data_ptr(), n_pages, at.data_ptr(), ko.data_ptr(), ko.stride(0), vo.data_ptr(), vo.stride(0), int(out_dtype == torch.bfloat16), heads, dk, dv, rows,
                               stream()))
        torch.cuda.synchronize()
        for out, want, d in ((ko, ref.read(cache, [s for _, s in live], dk, dv)[0], dk), (vo, ref.read(cache, [s for _, s in live], dk, dv)[1], dv)):
            expect = torch.full((rows, heads * d + pad), -5.0, dtype=out_dtype)
            for (i, _), t in zip(live, want):
                expect[i, :heads * d] = torch.tensor(t.reshape(-1)).to(out_dtype)
            assert torch.equal(out.cpu().nan_to_num(nan=-99.0), expect.nan_to_num(nan=-99.0))


@pytest.mark.parametrize("off", [1, 2, 4])
def test_rows_that_begin_anywhere(off):
    rng = np.random.default_rng(off)
    rows, heads, d, n_pages = 11, 2, 64, 2
    k, v = numbers((rows, heads, d), rng), numbers((rows, heads, d), rng)
    flat = [torch.zeros(off + rows * heads * d, device="cuda") for _ in range(2)]
    for f, t in zip(flat, (k, v)):
        f[off:] = torch.tensor(t.reshape(-1), device="cuda")
    kv, at = torch.zeros(n_pages, heads, ref.block_bytes(d, d), device="cuda", dtype=torch.uint8), dev(np.arange(rows) + 60)
    ok(lumi_b200.lib().lumi_k_kv4_append(flat[0][off:].data_ptr(), heads * d, flat[1][off:].data_ptr(), heads * d, 0, at.data_ptr(), kv.data_ptr(), n_pages, heads, d, d, rows, stream()))
    got = ref.read(kv.cpu().numpy(), np.arange(rows) + 60, d, d)
    for g, t in zip(got, (k, v)):
        assert np.array_equal(g, ref.values(*ref.quantise(t)))


def test_pointers_of_the_host_are_refused():
    host = torch.zeros(1024)
    there = torch.zeros(1 << 16, device="cuda", dtype=torch.uint8)
    lib = lumi_b200.lib()
    assert lib.lumi_k_kv4_append(host.data_ptr(), 64, there.data_ptr(), 64, 0, there.data_ptr(), there.data_ptr(), 1, 1, 64, 64, 1, stream()) == -1
    assert lib.lumi_k_page_plan(host.data_ptr(), *[there.data_ptr()], 1, there.data_ptr(), 1, there.data_ptr(), 1, *[there.data_ptr()] * 6, 1, stream()) == -1
